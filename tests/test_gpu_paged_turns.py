"""Paged KV cache on the GPU: reads whose workgroups have several units of work, and
reads and appends of more rows than one turn of the largest grid takes."""
import numpy as np
import pytest
import torch

from paged_common import DTYPE, i32

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def rng_of(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


# A read has at most 16384 workgroups; a unit is 64, 32, 16 or 8 rows of head dims up to 64, 128, 256, 512.
READS = [(300, 8, 8, 16, 3000), (131, 4, 128, 48, 4096), (70, 3, 512, 32, 2500)]
# Turns of a grid of 2^20 workgroups: 4 rows each (append and read), 32 of 8.
TURNS = [(2, 4, 1100003), (8, 64, 262201)]


def random_kv(fmt, n_pages, hkv, page, d, seed):
    from bitnetrs_amd import PagedKV

    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (n_pages, hkv, page, d)

    def codes():
        if fmt == "int8":
            return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        x = torch.randn(shape, generator=g, device="cuda")
        return (x * 100).to(DTYPE[fmt]) if fmt == "fp8" else x.to(DTYPE[fmt])

    sc = [None, None]
    if fmt in ("fp8", "int8"):
        sc = [torch.rand(shape[:3], generator=g, device="cuda") + 0.01 for _ in range(2)]
    return PagedKV.from_tensors(codes(), codes(), *sc)


def same_bits(a, b):
    """Equal bits, NaN (an e4m3 code past 448) for NaN."""
    return torch.equal(a.nan_to_num(1e30, torch.inf, -torch.inf).contiguous().view(torch.int32),
                       b.nan_to_num(1e30, torch.inf, -torch.inf).contiguous().view(torch.int32))


def value_rows(kv, name, pages, rows):
    """[n, hkv, d] as fp32: one rounded product; zeros where there is no page."""
    at = pages.clamp_min(0)
    raw = getattr(kv, name)
    x = raw.view(torch.uint8)[at, :, rows].view(raw.dtype).float() if kv.fmt == "fp8" else raw[at, :, rows].float()
    s = getattr(kv, name + "_scales")
    if s is not None:
        x = x * s[at, :, rows][..., None]
    return torch.where((pages >= 0)[:, None, None], x, 0.0)


@pytest.mark.parametrize("starts", [False, True])
@pytest.mark.parametrize("batch,hkv,d,page,top", READS)
@pytest.mark.parametrize("fmt", ["f32", "bf16", "fp8", "int8"])
def test_read_shares_of_several_units(backend, fmt, batch, hkv, d, page, top, starts):
    """More units than workgroups, so that shares hold several, start and end inside
    sequences and cross heads and sequences; batches past 64, some sequences
    empty, some pages not there; bit for bit."""
    say(f"read shares {fmt} {batch} x {hkv}/{d} page {page} starts {starts}")
    rng = rng_of("shares", fmt, batch, d, starts)
    lens = rng.integers(0, top + 1, batch)
    lens[rng.choice(batch, batch // 10, replace=False)] = 0
    lens[batch // 2] = top
    first = rng.integers(0, top // 4, batch) if starts else np.zeros(batch, np.int64)
    width = -(-top // page)
    order = rng.permutation(batch * width).astype(np.int32).reshape(batch, width)
    order[rng.random(order.shape) < 0.02] = -1
    kv = random_kv(fmt, batch * width, hkv, page, d, batch + d)
    table = torch.from_numpy(order).cuda()
    out = [torch.full((batch, hkv, top, d), 9.0, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, table, i32(lens), *out, starts=i32(first) if starts else None)
    torch.cuda.synchronize()
    for name, o in zip("kv", out):
        for s in range(batch):
            t = torch.arange(first[s], max(lens[s], first[s]), device="cuda")
            want = value_rows(kv, name, table[s, t // page].long(), t % page).transpose(0, 1)
            n = len(t)
            assert same_bits(o[s, :, :n], want), (name, s)
            assert (o[s, :, n:] == 9.0).all(), (name, s)
    del out, kv
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d,hkv,n", TURNS)
def test_append_and_read_past_one_turn(backend, d, hkv, n):
    """More rows than the largest grid takes in one turn: codes, scales and the
    rows read back, bit for bit."""
    say(f"append {n} tokens of {hkv}/{d}")
    from bitnetrs_amd import PagedKV

    page = 64
    width = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(d)
    table = torch.randperm(width + 1, generator=g, device="cuda")[:width].int().view(1, width)
    x = [torch.randn(n, hkv, d, generator=g, device="cuda") for _ in range(2)]
    kv = PagedKV(width + 1, page, hkv, d, "int8")
    t = torch.arange(n, device="cuda")
    backend.dev_paged_append(kv, None, *x, None, t.int(), table, seqs=torch.zeros(n, dtype=torch.int32, device="cuda"))
    out = [torch.full((1, hkv, n + 1, d), 9.0, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, table, i32([n]), *out)
    torch.cuda.synchronize()
    pages = table[0, t // page].long()
    for name, rows, o in zip("kv", x, out):
        m = rows.abs().amax(-1, keepdim=True)
        top = torch.full_like(m, 127.0)
        codes, scales = (rows * (top / m)).round().to(torch.int8), (m / top)[..., 0]
        assert torch.equal(getattr(kv, name)[pages, :, t % page], codes), name
        assert torch.equal(getattr(kv, name + "_scales")[pages, :, t % page], scales), name
        assert torch.equal(o[0, :, :n], (codes.float() * scales[..., None]).transpose(0, 1)), name
        assert (o[0, :, n:] == 9.0).all(), name
    del x, out, kv
    torch.cuda.empty_cache()
