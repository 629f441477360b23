"""Paged KV cache on the GPU: append, read and decode attention against their
definitions (tests/paged_common.py), at the sizes, lengths and pages where
they can go wrong, and a run of the three as a server would use them."""
import numpy as np
import pytest
import torch

from paged_common import (DTYPE, FORMATS, Pool, attention, attention_bound, encode, i32, rotate,
                          values)

pytestmark = pytest.mark.gpu

THETA = 500000.0


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def rng_of(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


def same(a, b):
    """Equal bits, NaN for NaN."""
    a, b = np.ascontiguousarray(a, np.float32), np.ascontiguousarray(b, np.float32)
    both = np.isnan(a) & np.isnan(b)
    return np.array_equal(np.where(both, 0, a).view(np.uint32), np.where(both, 0, b).view(np.uint32))


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
SHAPES = [(20, 5, 128, 16), (8, 8, 64, 16), (14, 2, 80, 32), (4, 4, 96, 64), (16, 2, 256, 128),
          (3, 1, 2, 1), (2, 1, 6, 5), (6, 3, 34, 7), (4, 2, 130, 48), (5, 5, 510, 16), (2, 2, 512, 8)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,page", SHAPES)
def test_append(backend, fmt, hq, hkv, d, page):
    """Ragged tokens of three sequences in no order, with rotation: q_out, codes
    and scales bit by bit, and no other row of the pool touched."""
    say(f"append {fmt} {hq}/{hkv}/{d} page {page}")
    rng = rng_of(fmt, hq, hkv, d, page)
    width = -(-40 // page)
    pool = Pool(rng, fmt, [width * page] * 3, hkv, d, page)
    where = [(s, t) for s, t0, n in ((0, 0, 5), (1, 11, 21), (2, 39, 1)) for t in range(t0, t0 + n)]
    rng.shuffle(where)
    seqs, pos = (np.array(x) for x in zip(*where))
    n = len(where)
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (hq, hkv, hkv))
    cos, sin = backend.rope_table(width * page, d, THETA)
    cosn, sinn = cos.cpu().numpy(), sin.cpu().numpy()
    kv = pool.device()
    q_out = torch.full((n, hq, d), 7.0, device="cuda")
    backend.dev_paged_append(kv, torch.from_numpy(q).cuda(), torch.from_numpy(k).cuda(),
                             torch.from_numpy(v).cuda(), q_out, i32(pos), i32(pool.table), cos, sin,
                             seqs=i32(seqs))
    torch.cuda.synchronize()
    assert same(q_out.cpu(), rotate(q, cosn[pos], sinn[pos]))
    for name, rows in (("k", rotate(k, cosn[pos], sinn[pos])), ("v", v)):
        codes, scales = encode(rows, fmt)
        want, want_s = pool.codes[name].clone(), pool.scales[name]
        want_s = None if want_s is None else want_s.copy()
        pages = pool.table[seqs, pos // page]
        raw = torch.uint8
        want.view(raw)[torch.from_numpy(pages).long(), :, torch.from_numpy(pos % page)] = codes.view(raw)
        got = getattr(kv, name).cpu()
        assert torch.equal(got.view(raw), want.view(raw)), name
        if want_s is not None:
            want_s[pages, :, pos % page] = scales
            assert same(getattr(kv, name + "_scales").cpu(), want_s), name


def test_append_rotation_is_rope_embed(backend):
    """With rope_table's tables the rotation has rope_embed's bits, far out too."""
    d, hq, hkv = 128, 20, 5
    rng = rng_of("rope")
    cos, sin = backend.rope_table(9000, d, THETA)
    pos = np.array([0, 1, 4095, 4096, 8999])
    q, k = (rng.standard_normal((5, h, d)).astype(np.float32) for h in (hq, hkv))
    kv = Pool(rng, "f32", [9008] * 5, hkv, d, 16)
    pool = kv.device()
    q_out = torch.empty(5, hq, d, device="cuda")
    tk = torch.from_numpy(k).cuda()
    backend.dev_paged_append(pool, torch.from_numpy(q).cuda(), tk, tk, q_out, i32(pos), i32(kv.table),
                             cos, sin)
    got = pool.k.cpu().numpy()
    for i, p in enumerate(pos):
        qi, ki = q[i].copy().reshape(-1), k[i].copy().reshape(-1)
        backend.rope_embed(qi, ki, int(p), d, hq, hkv, THETA)
        assert same(q_out[i].cpu().numpy().reshape(-1), qi)
        assert same(got[kv.table[i, p // 16], :, p % 16].reshape(-1), ki)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_without_rotation_or_q_in_place(backend, fmt):
    """No tables: rows as they are.  No q: nothing of it.  q_out may be q."""
    d, hq, hkv, page, n = 64, 6, 2, 16, 9
    rng = rng_of("plain", fmt)
    pool = Pool(rng, fmt, [n], hkv, d, page)
    x = torch.from_numpy(rng.standard_normal((n, hkv, d)).astype(np.float32)).cuda()
    kv = pool.device()
    args = dict(positions=i32(range(n)), block_table=i32(pool.table), seqs=i32([0] * n))
    backend.dev_paged_append(kv, None, x, x * 2, None, **args)
    want = values(*encode(x.cpu().numpy(), fmt)), values(*encode((x * 2).cpu().numpy(), fmt))
    out = [torch.zeros(1, hkv, n, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, args["block_table"], i32([n]), *out)
    for o, w in zip(out, want):
        assert same(o[0].cpu().numpy().transpose(1, 0, 2), w)
    q = torch.from_numpy(rng.standard_normal((n, hq, d)).astype(np.float32)).cuda()
    keep = q.clone()
    cos, sin = backend.rope_table(n, d, THETA)
    backend.dev_paged_append(kv, q, x, x, q, cos=cos, sin=sin, **args)
    assert same(q.cpu(), rotate(keep.cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy()))
    before = keep.clone()
    backend.dev_paged_append(kv, keep, x, x, keep, **args)  # neither rotated nor changed
    assert torch.equal(keep, before)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,page", [(128, 16), (10, 3)])
def test_append_leaves_out(backend, fmt, d, page):
    """Padding tokens, positions and sequences outside the table, positions past
    the rotation's tables, pages that are not there: nothing written."""
    rng = rng_of("out", fmt, d)
    hq, hkv = 4, 2
    pool = Pool(rng, fmt, [4 * page] * 2, hkv, d, page)
    n_pages = pool.codes["k"].shape[0]
    pool.table[0, 1], pool.table[1, 2] = -1, n_pages
    cos, sin = backend.rope_table(3 * page + 1, d, THETA)
    #        good  pad  missing  past the table  past cos      no such page  bad sequences        good
    pos = [0, -1, page, 4 * page, 3 * page + 1, 2 * page, 1, 1, 1 << 30, 3 * page]
    seqs = [0, 0, 0, 0, 0, 1, 2, -1, 0, 1]
    good, q_only = [0, 9], [2, 5]
    n = len(pos)
    q, k = (torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).cuda() for h in (hq, hkv))
    q_out = torch.full_like(q, 7.0)
    kv = pool.device()
    backend.dev_paged_append(kv, q, k, k, q_out, i32(pos), i32(pool.table), cos, sin, seqs=i32(seqs))
    torch.cuda.synchronize()
    p = np.array(pos)
    cosn, sinn = cos.cpu().numpy(), sin.cpu().numpy()
    for i in range(n):
        if i in good + q_only:  # a page that is not there drops the rows, not the query
            assert same(q_out[i:i + 1].cpu(), rotate(q[i:i + 1].cpu().numpy(), cosn[p[i:i + 1]], sinn[p[i:i + 1]]))
        else:
            assert (q_out[i] == 7.0).all()
    want = pool.codes["v"].clone()
    codes, _ = encode(k.cpu().numpy(), fmt)
    for i in good:
        want.view(torch.uint8)[pool.table[seqs[i], pos[i] // page], :, pos[i] % page] = codes[i].view(torch.uint8)
    assert torch.equal(kv.v.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [128, 22])
def test_append_extreme_rows(backend, fmt, d):
    """Zeros, the largest and smallest floats, ties, infinities and NaN."""
    rng = rng_of("extreme", fmt, d)
    x = rng.standard_normal((12, 1, d)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-38)
    x[2] = np.float32(3.4e38) * np.sign(x[2])
    x[3, 0, 3] = np.inf
    x[4, 0, d - 1] = -np.inf
    x[5, 0, 0] = np.nan
    x[6] = np.float32(1e-45)
    x[7] = (np.arange(d) % 128) / np.float32(2)  # ties of int8, with the maximum below
    x[7, 0, 1] = 127
    x[8] = np.float32(2.0) ** (np.arange(d) % 40 - 20)
    x[9, 0, 1:] = 0
    x[10] = -0.0
    x[11] = np.nan
    pool = Pool(rng, fmt, [12], 1, d, 16)
    kv = pool.device()
    t = torch.from_numpy(x).cuda()
    backend.dev_paged_append(kv, None, t, t, None, i32(range(12)), i32(pool.table), seqs=i32([0] * 12))
    codes, scales = encode(x, fmt)
    out = [torch.zeros(1, 1, 12, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, i32(pool.table), i32([12]), *out)
    for o in out:
        assert same(o[0].cpu().numpy().transpose(1, 0, 2), values(codes, scales))


# ---------------------------------------------------------------------------
# read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,page", SHAPES)
def test_read(backend, fmt, hq, hkv, d, page):
    """Rows of ragged sequences, whole and from a start; what lies behind stays.
    Lengths of 0 and below, past the table, starts past the length and below
    0, pages that are not there (zeros)."""
    say(f"read {fmt} {hkv}/{d} page {page}")
    rng = rng_of("read", fmt, hkv, d, page)
    lens = [3 * page, 1, 0, 2 * page + 1 if page > 1 else 2, 3 * page, 2 * page]
    pool = Pool(rng, fmt, lens, hkv, d, page, width=3)
    pool.table[5, 0] = -5
    pool.table[4, 1] = 1 << 30
    kv = pool.device()
    asked = np.array([1 << 30, 1, -7, lens[3], lens[4], lens[5]])
    real = np.clip(asked, 0, 3 * page)
    for starts, cap in ((None, 3 * page), (None, max(1, page - 1)), ([1, 0, 0, 2, page, -1], 2 * page),
                        ([3 * page, 1, 5, 0, 0, 0], 3 * page + 5)):
        out = [torch.full((6, hkv, cap, d), 9.0, device="cuda") for _ in range(2)]
        backend.dev_paged_read(kv, i32(pool.table), i32(asked), *out,
                               starts=None if starts is None else i32(starts))
        torch.cuda.synchronize()
        for name, o in zip("kv", out):
            want = np.full((6, hkv, cap, d), 9.0, np.float32)
            for s in range(6):
                first = 0 if starts is None else starts[s]
                n = min(real[s] - first, cap)
                if first < 0 or n <= 0:
                    continue
                rows, there = pool.rows(name, s, real[s])
                rows = np.where(there[:, None, None], rows, 0)
                want[s, :, :n] = rows[first:first + n].transpose(1, 0, 2)
            assert same(o.cpu(), want), (name, starts, cap)


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
def check_decode(backend, pool, hq, q=None, lens=None, kv=None, workspace=None, times=1):
    kv = kv or pool.device()
    lens = pool.lens if lens is None else lens
    B, d = len(lens), pool.d
    rng = rng_of("q", hq, d, B)
    q = rng.standard_normal((B, hq, d)).astype(np.float32) if q is None else q
    ws = backend.paged_workspace(kv, B, hq) if workspace is None else workspace
    out = torch.full((B, hq, d), float("nan"), device="cuda")
    table, tl, tq = i32(pool.table), i32(lens), torch.from_numpy(q).cuda()
    for _ in range(times):
        backend.dev_paged_decode_attention(kv, tq, table, tl, out, ws)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    for s in range(B):
        n = int(np.clip(lens[s], 0, pool.table.shape[1] * pool.page))
        (k, there), (v, _) = pool.rows("k", s, n), pool.rows("v", s, n)
        k, v = k[there], v[there]
        ref, mag, size = attention(q[s], k, v)
        if not len(k):
            assert (got[s] == 0).all(), f"sequence {s} without a row"
            continue
        err, room = np.abs(got[s] - ref), attention_bound(len(k), d, mag, size)
        assert (err <= room).all(), (f"sequence {s}, {len(k)} rows: off by {err.max():.3g}, "
                                     f"{(err / room).max():.3g} of the bound")
    return out


RAGGED = [1, 0, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 500, 1, 1000]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,page", SHAPES + [(16, 1, 128, 16), (16, 1, 256, 16), (17, 1, 64, 16), (40, 2, 48, 32),
                                                    (2, 2, 16, 16), (6, 2, 192, 16), (1, 1, 128, 64),
                                                    (12, 4, 128, 48), (9, 3, 112, 16)])
def test_decode(backend, fmt, hq, hkv, d, page):
    """Ragged batches: lengths of nothing, one, around tiles and pages."""
    say(f"decode {fmt} {hq}/{hkv}/{d} page {page}")
    pool = Pool(rng_of("decode", fmt, hkv, d, page), fmt, RAGGED, hkv, d, page, spread=0.3)
    check_decode(backend, pool, hq)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [7], [4096], [5001], [20000, 3], [0] * 70 + [300] + [0] * 60 + [5],
                                  [9000] + [1] * 200])
def test_decode_batches(backend, fmt, lens):
    """From one token to long sequences split over the card, batches past 64."""
    say(f"decode {fmt} lens {lens[:4]} x{len(lens)}")
    pool = Pool(rng_of("batches", fmt, len(lens), max(lens)), fmt, lens, 5, 128, 16, spread=0.3)
    check_decode(backend, pool, 20)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d,lens", [(12, 1, 80, [30000]), (16, 1, 128, [17, 21000]), (16, 1, 256, [9000]),
                                           (14, 2, 128, [12000, 3000]), (4, 1, 128, [40000]), (3, 1, 26, [9000])])
def test_decode_many_pieces(backend, fmt, hq, hkv, d, lens):
    """Items of many workgroups, joined in groups first, the last one not full;
    the same bits again on the used workspace."""
    say(f"decode many pieces {fmt} {hq}/{hkv}/{d} {lens}")
    pool = Pool(rng_of("many", fmt, hq, d), fmt, lens, hkv, d, 16, spread=0.3)
    kv = pool.device()
    ws = backend.paged_workspace(kv, 2, hq)
    first = check_decode(backend, pool, hq, kv=kv, workspace=ws)
    assert (ws[:1536 * 256] == 0).all()
    assert torch.equal(first, check_decode(backend, pool, hq, kv=kv, workspace=ws, times=3))


@pytest.mark.parametrize("fmt,page", [("int8", 16), ("bf16", 48), ("f32", 64), ("fp8", 128)])
def test_decode_long_pieces(backend, fmt, page):
    """Pieces of more than 4096 rows of one workgroup, with pages that are not
    there among them and a last page that is not full."""
    say(f"decode long pieces {fmt}")
    rng = rng_of("long", fmt)
    pool = Pool(rng, fmt, [150001], 16, 16, page, spread=0.3)
    pool.table[0, rng.choice(pool.table.shape[1], 40, replace=False)] = -1
    check_decode(backend, pool, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,page", [(128, 16), (128, 64), (80, 32), (10, 3)])
def test_decode_missing_pages_and_lengths(backend, fmt, d, page):
    """Pages that are not there leave their rows out; a sequence of only such
    pages has no row; lengths past the table and below 0."""
    say(f"decode missing {fmt} {d} page {page}")
    pool = Pool(rng_of("missing", fmt, d, page), fmt, [5 * page] * 6, 2, d, page, spread=0.3)
    n_pages = pool.codes["k"].shape[0]
    pool.table[0, 0] = -1
    pool.table[1, 4] = n_pages
    pool.table[2, 2] = -(1 << 31)
    pool.table[3, :] = -1
    pool.table[4, 1:4] = (1 << 31) - 1
    check_decode(backend, pool, 8, lens=[5 * page, 5 * page - 1, 1 << 30, 5 * page, 3 * page, -3])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (22, 5)])
def test_decode_ignores_what_is_not_attended(backend, fmt, d, page):
    """NaN and infinities behind the last row of a page, in unused pages, and in
    page 0 where a missing page might be read by mistake."""
    rng = rng_of("nan", fmt, d)
    lens = [page + 3, 1, 2 * page, 3 * page - 1]
    pool = Pool(rng, fmt, lens, 2, d, page, width=3, spread=0.3)
    used = set()
    for s, n in enumerate(lens):
        used |= {(int(pool.table[s, t // page]), t % page) for t in range(n)}
    bad = float("nan")
    for name in "kv":
        c = pool.codes[name].float()
        for pg in range(c.shape[0]):
            for r in range(page):
                if (pg, r) not in used:
                    c[pg, :, r] = bad if (pg + r) % 2 else float("inf") if fmt in ("f32", "bf16") else 127.0
                    if pool.scales[name] is not None:
                        pool.scales[name][pg, :, r] = bad
        pool.codes[name] = c.nan_to_num(0).to(DTYPE[fmt]) if fmt == "int8" else c.to(DTYPE[fmt])
    out = check_decode(backend, pool, 6)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,page", [(128, 16), (26, 4)])
def test_decode_scores_of_any_size(backend, fmt, d, page):
    """Scores far apart (one row takes all), all equal, huge and tiny values."""
    rng = rng_of("scores", fmt, d)
    pool = Pool(rng, fmt, [300, 77, 200, 300], 2, d, page, spread=0.3)
    q = rng.standard_normal((4, 4, d)).astype(np.float32)
    q[0] *= 300.0  # one row takes nearly all of the weight
    q[1] = 0.0  # all rows weigh the same
    q[2] *= np.float32(1e-20)
    q[3, 0] *= 30.0
    check_decode(backend, pool, 4, q=q)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("d,page", [(128, 16), (26, 4)])
def test_decode_scales_of_any_size(backend, fmt, d, page):
    """Rows whose scales differ by many powers of two, keys and values apart."""
    rng = rng_of("scales", fmt, d)
    pool = Pool(rng, fmt, [600, 130], 2, d, page, spread=0.1)
    pool.scales["v"] *= np.exp2(rng.integers(-40, 40, pool.scales["v"].shape)).astype(np.float32)
    pool.scales["k"] *= np.exp2(rng.integers(-12, 1, pool.scales["k"].shape)).astype(np.float32)
    check_decode(backend, pool, 8)


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_non_finite_rows_show(backend, fmt):
    """An attended row that is not finite makes its outputs non-finite, and only
    those of its kv head."""
    pool = Pool(rng_of("show", fmt), fmt, [100], 2, 128, 16, spread=0.3)
    pg, r = int(pool.table[0, 3]), 5
    if fmt in ("f32", "bf16"):
        pool.codes["k"][pg, 0, r, 9] = float("nan")
    else:
        pool.scales["k"][pg, 0, r] = float("nan")
    kv = pool.device()
    q = torch.randn(1, 8, 128, device="cuda")
    out = torch.zeros_like(q)
    backend.dev_paged_decode_attention(kv, q, i32(pool.table), i32([100]), out,
                                       backend.paged_workspace(kv, 1, 8))
    assert not torch.isfinite(out[0, :4]).any() and torch.isfinite(out[0, 4:]).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_same_bits_and_workspace_left_ready(backend, fmt):
    """The same call has the same bits every time, on a used workspace, after a
    call of other sizes on it, and its tickets are zero in between."""
    pool = Pool(rng_of("bits", fmt), fmt, [7000, 130, 0, 2500], 5, 128, 16, spread=0.3)
    small = Pool(rng_of("bits2", fmt), fmt, [600], 5, 128, 16, spread=0.3)
    kv, kv2 = pool.device(), small.device()
    ws = backend.paged_workspace(kv, 4, 20)
    first = check_decode(backend, pool, 20, kv=kv, workspace=ws)
    assert (ws[:1536 * 256] == 0).all()
    check_decode(backend, small, 20, kv=kv2, workspace=ws)
    again = check_decode(backend, pool, 20, kv=kv, workspace=ws, times=4)
    assert torch.equal(first, again)


def test_workspace_of_many_shapes(backend):
    """One workspace for calls of other batches, heads, groups and kernels in
    turn, each leaving pieces of its own: none finds another's tickets."""
    shapes = [([900] * 16, 16, 16, 64, 16), ([5000], 16, 16, 64, 16), ([3000, 10] * 8, 32, 2, 128, 16),
              ([700] * 9, 4, 4, 26, 5), ([900] * 40, 16, 16, 64, 16), ([2000], 5, 5, 128, 48)]
    pools = [Pool(rng_of("shapes", i), "bf16", lens, hkv, d, page, spread=0.3)
             for i, (lens, _, hkv, d, page) in enumerate(shapes)]
    kvs = [p.device() for p in pools]
    ws = max((backend.paged_workspace(kv, len(s[0]), s[1]) for kv, s in zip(kvs, shapes)), key=len)
    for turn in range(2):
        for p, kv, s in zip(pools, kvs, shapes):
            check_decode(backend, p, s[1], kv=kv, workspace=ws)


@pytest.mark.parametrize("fmt", FORMATS)
def test_unaligned_buffers(backend, fmt):
    """Pools, queries and outputs that start off a 16-byte boundary."""
    rng = rng_of("unaligned", fmt)
    pool = Pool(rng, fmt, [70, 33], 2, 64, 16, spread=0.3)
    from bitnetrs_amd import PagedKV

    def off(t):
        raw = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        raw[1:].view(torch.uint8).copy_(t.reshape(-1).view(torch.uint8).cuda())
        return raw[1:].view(t.shape)

    sc = [None if pool.scales[n] is None else off(torch.from_numpy(pool.scales[n])) for n in "kv"]
    kv = PagedKV.from_tensors(off(pool.codes["k"]), off(pool.codes["v"]), *sc)
    check_decode(backend, pool, 6, kv=kv)
    q = off(torch.from_numpy(rng.standard_normal((2, 6, 64)).astype(np.float32)))
    x = off(torch.from_numpy(rng.standard_normal((2, 2, 64)).astype(np.float32)))
    q_out = off(torch.zeros(2, 6, 64))
    cos, sin = backend.rope_table(80, 64, THETA)
    backend.dev_paged_append(kv, q, x, x, q_out, i32([5, 6]), i32(pool.table), off(cos), off(sin))
    c, s = cos[[5, 6]].cpu().numpy(), sin[[5, 6]].cpu().numpy()
    assert same(q_out.cpu(), rotate(q.cpu().numpy(), c, s))
    out = [off(torch.zeros(2, 2, 1, 64)) for _ in range(2)]
    backend.dev_paged_read(kv, i32(pool.table), i32([6, 7]), *out, starts=i32([5, 6]))
    assert same(out[0][:, :, 0].cpu(), values(*encode(rotate(x.cpu().numpy(), c, s), fmt)))
    assert same(out[1][:, :, 0].cpu(), values(*encode(x.cpu().numpy(), fmt)))


@pytest.mark.parametrize("fmt,d", [("int8", 128), ("int8", 90), ("f32", 128)])
def test_offsets_past_32_bits(backend, fmt, d):
    """Rows in pages whose first element is past 2^31 (bytes past 2^32 for f32)."""
    page, hkv, hq, n = 64, 4, 8, 150
    n_pages = (1 << 31) // (page * hkv * d) + 40
    say(f"pool of {n_pages} pages, {fmt} {d}")
    from bitnetrs_amd import PagedKV

    kv = PagedKV(n_pages, page, hkv, d, fmt)
    rng = rng_of("far", d)
    table = i32([[n_pages - 3, 2, n_pages - 1]])
    x = [torch.from_numpy(rng.standard_normal((n, hkv, d)).astype(np.float32)).cuda() for _ in range(2)]
    backend.dev_paged_append(kv, None, *x, None, i32(range(n)), table, seqs=i32([0] * n))
    out = [torch.zeros(1, hkv, n, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, table, i32([n]), *out)
    k, v = (values(*encode(t.cpu().numpy(), fmt)) for t in x)
    for o, w in zip(out, (k, v)):
        assert same(o[0].cpu().numpy().transpose(1, 0, 2), w)
    q = rng.standard_normal((1, hq, d)).astype(np.float32)
    got = torch.zeros(1, hq, d, device="cuda")
    backend.dev_paged_decode_attention(kv, torch.from_numpy(q).cuda(), table, i32([n]), got,
                                       backend.paged_workspace(kv, 1, hq))
    ref, mag, size = attention(q[0], k, v)
    assert (np.abs(got[0].cpu().numpy() - ref) <= attention_bound(n, d, mag, size)).all()
    del kv, out
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
def test_serving_run(backend, fmt):
    """As a server uses them: prompts appended, read back into the contiguous
    layout and attended by the prefill; then tokens decoded one by one, two
    sequences of different lengths at once, from a captured graph that replays
    with positions and lengths moved on the device; every step against 64
    bits, and in f32 against the contiguous decode too."""
    hq, hkv, d, page, width = 20, 5, 128, 16, 12
    rng = rng_of("serve", fmt)
    from bitnetrs_amd import PagedKV

    kv = PagedKV(2 * width + 1, page, hkv, d, fmt)
    order = rng.permutation(2 * width + 1)[:2 * width].reshape(2, width)
    table = i32(order)
    cos, sin = backend.rope_table(width * page, d, THETA)
    cosn, sinn = cos.cpu().numpy(), sin.cpu().numpy()
    prompts = [70, 33]
    hist = [[np.zeros((0, hkv, d), np.float32)] * 2 for _ in prompts]  # the rows that the cache stands for
    pos = np.concatenate([np.arange(n) for n in prompts])
    seqs = np.repeat([0, 1], prompts)
    q, k, v = (rng.standard_normal((len(pos), h, d)).astype(np.float32) for h in (hq, hkv, hkv))
    q_rot = torch.empty(len(pos), hq, d, device="cuda")
    backend.dev_paged_append(kv, *(torch.from_numpy(x).cuda() for x in (q, k, v)), q_rot, i32(pos), table,
                             cos, sin, seqs=i32(seqs))
    kr = values(*encode(rotate(k, cosn[pos], sinn[pos]), fmt))
    vr = values(*encode(v, fmt))
    for s in range(2):
        hist[s] = [kr[seqs == s], vr[seqs == s]]
    cap = max(prompts)
    kc, vc = (torch.zeros(2, hkv, cap, d, device="cuda") for _ in range(2))
    backend.dev_paged_read(kv, table, i32(prompts), kc, vc)
    for s, n in enumerate(prompts):
        out = torch.empty(n, hq, d, device="cuda")
        backend.dev_prefill_attention(q_rot[torch.from_numpy(seqs == s)].contiguous(), kc[s], vc[s], cap, out, n, 0, hq,
                                      hkv, d)
        got = out.cpu().numpy()
        qr = rotate(q[seqs == s], cosn[:n], sinn[:n])
        for t in (0, n // 2, n - 1):
            ref, mag, size = attention(qr[t], hist[s][0][:t + 1], hist[s][1][:t + 1])
            # the prefill's own rounding is the contiguous path's, held there to 1e-4 of the output
            assert (np.abs(got[t] - ref) <= attention_bound(t + 1, d, mag, size) + 1e-4 * np.abs(ref).max()).all()

    # decode: one graph, replayed with other inputs
    tq, tk, tv = (torch.zeros(2, h, d, device="cuda") for h in (hq, hkv, hkv))
    tpos, tlen = i32(prompts), i32([n + 1 for n in prompts])
    q_out, out = torch.zeros_like(tq), torch.zeros_like(tq)
    ws = backend.paged_workspace(kv, 2, hq)
    scratch = PagedKV(2 * width + 1, page, hkv, d, fmt)  # the warm-up writes elsewhere

    def step(pool):
        backend.dev_paged_append(pool, tq, tk, tv, q_out, tpos, table, cos, sin)
        backend.dev_paged_decode_attention(pool, q_out, table, tlen, out, ws)

    step(scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kv)
        tpos += 1
        tlen += 1
    for i in range(40):
        new = [rng.standard_normal((2, h, d)).astype(np.float32) for h in (hq, hkv, hkv)]
        for t, x in zip((tq, tk, tv), new):
            t.copy_(torch.from_numpy(x))
        graph.replay()
        torch.cuda.synchronize()
        at = np.array([n + i for n in prompts])
        qr = rotate(new[0], cosn[at], sinn[at])
        kr = values(*encode(rotate(new[1], cosn[at], sinn[at]), fmt))
        vr = values(*encode(new[2], fmt))
        got = out.cpu().numpy()
        for s in range(2):
            hist[s] = [np.concatenate([h, x[s:s + 1]]) for h, x in zip(hist[s], (kr, vr))]
            ref, mag, size = attention(qr[s], *hist[s])
            assert (np.abs(got[s] - ref) <= attention_bound(len(hist[s][0]), d, mag, size)).all(), (i, s)
        if i % 13 == 0:  # eager work in between, on the graph's own buffers
            eager = torch.zeros_like(out)
            backend.dev_paged_decode_attention(kv, q_out, table, i32(at + 1), eager, ws)
            assert torch.equal(eager, out)
    if fmt == "f32":  # the contiguous decode over the same rows
        n = len(hist[0][0])
        kc, vc = (torch.zeros(2, hkv, n, d, device="cuda") for _ in range(2))
        backend.dev_paged_read(kv, table, i32([n, n]), kc, vc)
        ref = torch.zeros(hq, d, device="cuda")
        backend.dev_decode_attention(q_out[0].contiguous(), kc[0], vc[0], n, ref, hq, hkv, d, n - 1)
        _, mag, size = attention(qr[0], *hist[0])
        assert (np.abs((out[0] - ref).cpu().numpy()) <= 2 * attention_bound(n, d, mag, size)).all()
    del graph


def test_two_streams_with_their_own_workspaces(backend):
    """Calls on two streams at once, each on its own workspace."""
    pools = [Pool(rng_of("streams", i), f, [6000, 900], 5, 128, 16, spread=0.3)
             for i, f in enumerate(("bf16", "int8"))]
    kvs = [p.device() for p in pools]
    q = torch.randn(2, 20, 128, device="cuda")
    tabs, lens = [i32(p.table) for p in pools], i32([6000, 900])
    ws = [backend.paged_workspace(kv, 2, 20) for kv in kvs]
    outs = [[torch.zeros_like(q) for _ in range(8)] for _ in pools]
    ref = []
    for kv, t, w in zip(kvs, tabs, ws):
        o = torch.zeros_like(q)
        backend.dev_paged_decode_attention(kv, q, t, lens, o, w)
        ref.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pools]
    for i in range(8):
        for j, s in enumerate(streams):
            backend.dev_paged_decode_attention(kvs[j], q, tabs[j], lens, outs[j][i], ws[j], stream=s)
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, ref[j]) for o in outs[j])


def test_two_graphs(backend):
    """Two captured calls, replayed in turn on one workspace, and side by side on
    two streams with a workspace each; eager work between the replays."""
    pools = [Pool(rng_of("graphs", i), f, lens, 5, 128, 16, spread=0.3)
             for i, (f, lens) in enumerate((("fp8", [5000, 700]), ("f32", [3000])))]
    kvs = [p.device() for p in pools]
    tabs, lens = [i32(p.table) for p in pools], [i32(p.lens) for p in pools]
    qs = [torch.randn(len(p.lens), 20, 128, device="cuda") for p in pools]
    refs, outs = ([torch.zeros_like(q) for q in qs] for _ in range(2))
    for shared in (True, False):
        ws = [backend.paged_workspace(kv, 2, 20) for kv in kvs]
        if shared:
            ws = [max(ws, key=len)] * 2
        graphs = []
        for i in range(2):
            backend.dev_paged_decode_attention(kvs[i], qs[i], tabs[i], lens[i], refs[i], ws[i])
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                backend.dev_paged_decode_attention(kvs[i], qs[i], tabs[i], lens[i], outs[i], ws[i])
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(4):
            for o in outs:
                o.fill_(float("nan"))
            torch.cuda.synchronize()
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(streams[0] if shared else s):
                    g.replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert torch.equal(outs[i], refs[i]), (shared, i)
            check_decode(backend, pools[1], 20, kv=kvs[1], workspace=ws[1])
        del graphs


def test_two_threads(backend):
    """Calls of two host threads at once, each on its own stream and workspace."""
    import threading

    pools = [Pool(rng_of("threads", i), f, [4000, 900, 30], 5, 128, 16, spread=0.3)
             for i, f in enumerate(("bf16", "int8"))]
    kvs = [p.device() for p in pools]
    tabs, lens = [i32(p.table) for p in pools], i32([4000, 900, 30])
    q = torch.randn(3, 20, 128, device="cuda")
    ws = [backend.paged_workspace(kv, 3, 20) for kv in kvs]
    outs = [[torch.zeros_like(q) for _ in range(20)] for _ in pools]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            for o in outs[i]:
                backend.dev_paged_decode_attention(kvs[i], q, tabs[i], lens, o, ws[i], stream=streams[i])
            with pytest.raises(TypeError):  # an error of this thread's own
                backend.dev_paged_decode_attention(kvs[i], q.cpu(), tabs[i], lens, o, ws[i])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for i in range(2):
        ref = torch.zeros_like(q)
        backend.dev_paged_decode_attention(kvs[i], q, tabs[i], lens, ref, ws[i])
        torch.cuda.synchronize()
        assert all(torch.equal(o, ref) for o in outs[i])


def test_python_refusals(backend):
    """Wrong shapes, types, layouts and devices are refused before the library."""
    from bitnetrs_amd import InvalidShape, PagedKV

    kv = PagedKV(4, 16, 2, 64, "int8")
    q, x = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")
    pos, table, lens = i32([0, 1, 2]), i32([[0, 1]] * 3), i32([1, 1, 1])
    ws = backend.paged_workspace(kv, 3, 4)
    out = torch.zeros_like(q)
    for args, error in (((q, x, x, out, pos.long(), table), TypeError), ((q, x, x[:2], out, pos, table), InvalidShape),
                        ((q, x, x, None, pos, table), TypeError), ((q.double(), x, x, out, pos, table), TypeError),
                        ((q, x.transpose(0, 1).contiguous().transpose(0, 1), x, out, pos, table), TypeError),
                        ((q, x, x.cpu(), out, pos, table), TypeError)):
        with pytest.raises(error):
            backend.dev_paged_append(kv, *args)
    for args, error in (((q[:2], table, lens, out, ws), InvalidShape), ((q, table, lens[:2], out, ws), InvalidShape),
                        ((q, table, lens, out, ws[:64]), InvalidShape), ((q, table, lens, out, ws.float()), TypeError),
                        ((q[:, :3].contiguous(), table, lens, out[:, :3].contiguous(), ws),
                         __import__("bitnetrs_amd").InvalidConfig)):
        with pytest.raises(error):
            backend.dev_paged_decode_attention(kv, *args)
    ko = torch.zeros(3, 2, 8, 64, device="cuda")
    for args, error in (((table, lens, ko, ko[:, :, :4].contiguous()), InvalidShape),
                        ((table, lens, ko[:, :1].contiguous(), ko), InvalidShape)):
        with pytest.raises(error):
            backend.dev_paged_read(kv, *args)
    for call, args in ((backend.dev_paged_append, (q, x, x, out, pos, lens)), (backend.dev_paged_read, (lens, lens, ko, ko)),
                       (backend.dev_paged_read, (table, lens, ko[0], ko[0])),
                       (backend.dev_paged_decode_attention, (q[0], table, lens, out, ws)),
                       (backend.dev_paged_decode_attention, (q, table, lens, out, ws.view(1, -1)))):
        with pytest.raises(InvalidShape):
            call(kv, *args)


def test_rope_table_leaves_the_contexts_own(backend):
    """A captured step of the contiguous cache still reads its table after
    tables of other sizes, head dims and thetas were built for paged caches."""
    d, hq, hkv, cap = 128, 20, 5, 4096
    q, k, v = (torch.randn(h * d, device="cuda") for h in (hq, hkv, hkv))
    kc, vc = (torch.randn(hkv, cap, d, device="cuda") for _ in range(2))
    out, ref = torch.zeros(hq * d, device="cuda"), torch.zeros(hq * d, device="cuda")
    args = (q, k, v, 70, hq, hkv, d, THETA, kc, vc, cap)
    backend.dev_decode_step(*args, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.dev_decode_step(*args, out)
    for n, dim, theta in ((20000, d, THETA), (100, 64, THETA), (5000, d, 1e4)):
        cos, sin = backend.rope_table(n, dim, theta)
        assert cos.shape == sin.shape == (n, dim // 2) and (cos[0] == 1).all() and (sin[0] == 0).all()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (out - ref).abs().max() <= 1e-5 * ref.abs().max()
    del graph


@pytest.mark.parametrize("hq,hkv,d,page", [(64, 1, 512, 16), (71, 1, 64, 16), (16, 1, 256, 16), (20, 1, 128, 8),
                                           (12, 2, 130, 16), (5, 5, 48, 32)])
def test_workspace_is_enough(backend, hq, hkv, d, page):
    """Long sequences in many pieces: nothing is written behind the workspace's bytes."""
    say(f"workspace {hq}/{hkv}/{d} page {page}")
    pool = Pool(rng_of("enough", hq, d), "bf16", [7000, 1200], hkv, d, page, spread=0.3)
    kv = pool.device()
    n = backend.paged_workspace(kv, 2, hq).numel()
    raw = torch.zeros(n + (1 << 20), dtype=torch.uint8, device="cuda")
    raw[n:] = 0x5A
    for _ in range(2):
        check_decode(backend, pool, hq, kv=kv, workspace=raw[:n])
    assert (raw[n:] == 0x5A).all() and (raw[:1536 * 256] == 0).all()


def test_rope_table_is_refused_under_capture(backend):
    """Its copies start in host memory that the call frees; the capture goes on."""
    from bitnetrs_amd import BackendError

    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(BackendError, match="capture"):
            backend.rope_table(16, 64, THETA)
        x += 1
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (x == 2 * (i + 1)).all()
    cos, _ = backend.rope_table(16, 64, THETA)
    assert (cos[0] == 1).all()
    del graph
