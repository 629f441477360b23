"""Paged KV cache on the GPU: every row of a long sequence counts once, with sums
that are exact, or nearly, in fp32 (tests/paged_rows.py)."""
import pytest
import torch

from paged_common import i32
from paged_rows import LONG, LONG_SHAPE, MANY, CountedPool

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def check_counted(backend, pool, hq, times=1):
    kv = pool.device()
    tq, table, lens = pool.queries(hq).cuda(), pool.table.cuda(), i32(pool.lens)
    ws = backend.paged_workspace(kv, len(pool.lens), hq)
    out = torch.full_like(tq, float("nan"))
    for _ in range(times):
        backend.dev_paged_decode_attention(kv, tq, table, lens, out, ws)
    torch.cuda.synchronize()
    got, g = out.cpu().double(), hq // pool.hkv
    for s in range(len(pool.lens)):
        want, room = pool.expected(s, hq)
        for j in range(g):
            sign = (torch.arange(pool.hkv) + j) % 2
            i = torch.arange(pool.hkv)
            err = (got[s, j::g] - want[sign, i]).abs()
            bad = err > room[sign, i]
            assert not bad.any(), (f"sequence {s}, query {j} of kv head {int(bad.any(-1).nonzero()[0])}: "
                                   f"off by {err.max():.3g}, room {room.max():.3g}")


@pytest.mark.parametrize("page,missing", LONG)
@pytest.mark.parametrize("fmt", ["f32", "bf16", "fp8", "int8"])
def test_every_row_of_long_pieces(backend, fmt, page, missing):
    say(f"rows of long pieces {fmt} page {page}")
    check_counted(backend, CountedPool(page, fmt, *LONG_SHAPE, page, missing), 512)


@pytest.mark.parametrize("hq,hkv,d,page,lens", MANY)
@pytest.mark.parametrize("fmt", ["f32", "bf16", "fp8", "int8"])
def test_every_row_of_many_pieces(backend, fmt, hq, hkv, d, page, lens):
    """Items of many workgroups, joined at once and in groups, on the matrix cores
    and (17 heads, odd pages, head dimensions) by the other kernel."""
    say(f"rows of many pieces {fmt} {hq}/{hkv}/{d} page {page} {lens[:3]}")
    check_counted(backend, CountedPool(hq, fmt, lens, hkv, d, page, 2), hq, times=2)
