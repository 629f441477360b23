"""Paged KV cache on the GPU: keys whose score is -infinity."""
import numpy as np
import pytest
import torch

from paged_common import Pool, attention, attention_bound, i32

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def rng_of(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 48), (26, 4), (256, 5)])
def test_decode_key_of_minus_infinity(backend, fmt, d, page, aligned):
    """A row whose score is -infinity has no weight, in any of the kernels and
    whatever bits the query has; a query with no other row gives zeros."""
    say(f"decode -inf keys {fmt} {d} page {page} aligned {aligned}")
    from bitnetrs_amd import PagedKV

    hq, hkv, lens = 6, 2, [150, 40, 33]
    rng = rng_of("inf", fmt, d, page)
    pool = Pool(rng, fmt, lens, hkv, d, page, spread=0.3)
    out_rows = {0: [0, 3, 17, 64, 149], 1: range(40), 2: [32]}
    for s, rows in out_rows.items():
        for t in rows:
            row = pool.codes["k"][int(pool.table[s, t // page]), 0, t % page]
            row[:] = torch.where(torch.from_numpy(rng.random(d) < 0.5), row, -torch.inf)
            row[t % d] = -torch.inf
    # queries above zero, so that each -infinity in a key is one in its score; some of them
    # powers of two once they are divided by sqrt(d) and turned to base 2
    q = np.abs(rng.standard_normal((3, hq, d)).astype(np.float32)) + np.float32(0.1)
    scale = np.float32(1.4426950408889634 / np.sqrt(np.float64(d)))
    one = next(x for x in np.float32(1) / scale * (1 + np.arange(-8, 9, dtype=np.float32) * np.float32(2.0 ** -24))
               if np.float32(x) * scale == 1)
    q[:, 0::3] = one
    q[:, 1::3, ::2] = one / 2
    kv = pool.device()
    tq = torch.from_numpy(q).cuda()
    if not aligned:  # the queries start off a 16-byte boundary
        raw = torch.zeros(q.size + 1, device="cuda")
        raw[1:] = tq.reshape(-1)
        tq = raw[1:].view(q.shape)
    out = torch.full(q.shape, float("nan"), device="cuda")
    backend.dev_paged_decode_attention(kv, tq, i32(pool.table), i32(lens), out, backend.paged_workspace(kv, 3, hq))
    got = out.cpu().numpy()
    g = hq // hkv
    for s, n in enumerate(lens):
        (k, _), (v, _) = pool.rows("k", s, n), pool.rows("v", s, n)
        for h in range(hkv):
            keep = np.array([h > 0 or t not in out_rows[s] for t in range(n)])
            ref, mag, size = attention(q[s, h * g:(h + 1) * g], k[keep, h:h + 1], v[keep, h:h + 1])
            x = got[s, h * g:(h + 1) * g]
            if not keep.any():
                assert (x == 0).all(), (s, h)
            else:
                assert (np.abs(x - ref) <= attention_bound(int(keep.sum()), d, mag, size)).all(), (s, h)
