"""The paged cache's 4-bit format without a GPU: its definition, and what is
refused."""
import numpy as np
import pytest
import torch

import bitnetrs_amd
from bitnetrs_amd import _lib
from fp4_common import E2M1, TINY, encode, values
from test_paged import append, decode, desc, read, workspace, P
from common import error_from_parts

CALLS = [append, read, decode]


def fp4(**kw):
    return desc(**dict(dict(format=_lib.BNR_KV_FP4), **kw))


@pytest.mark.parametrize("bad,kind,text", [
    (dict(k_scales=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(v_scales=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(head_dim=63), _lib.BNR_INVALID_CONFIG, "head_dim"),
    (dict(head_dim=514), _lib.BNR_INVALID_CONFIG, "head_dim"),
    (dict(n_pages=0), _lib.BNR_INVALID_SHAPE, "n_pages"),
])
@pytest.mark.parametrize("call", CALLS)
def test_bad_pool_is_refused(call, bad, kind, text):
    assert call(fp4(**bad)) == kind
    assert text in error_from_parts()[1]


def test_workspace_is_that_of_the_shape():
    for d, page, heads in ((64, 16, 4), (128, 16, 32), (80, 5, 6)):
        a = workspace(fp4(head_dim=d, page_size=page), n_heads=heads)
        assert a[0] == _lib.BNR_OK and a == workspace(desc(head_dim=d, page_size=page), n_heads=heads)
    assert workspace(fp4(format=6))[0] == _lib.BNR_INVALID_CONFIG


def test_nothing_to_do_is_no_error():
    assert append(fp4(), n_tokens=0) == _lib.BNR_OK
    assert read(fp4(), batch=0) == _lib.BNR_OK
    assert decode(fp4(k=P + 1, k_scales=P + 3), batch=0) == _lib.BNR_OK


@pytest.mark.parametrize("d", [2, 30, 32, 34, 80, 128, 512])
def test_pool_shapes(d):
    kv = bitnetrs_amd.PagedKV(3, 16, 5, d, "fp4", device="cpu")
    assert kv.fmt == "fp4" and kv.head_dim == d and kv.k.dtype == torch.uint8
    assert kv.k.shape == (3, 5, 16, d // 2) and kv.v_scales.shape == (3, 5, 16, -(-d // 32))
    same = bitnetrs_amd.PagedKV.from_tensors(kv.k, kv.v, kv.k_scales, kv.v_scales)
    assert (same.fmt, same.head_dim) == ("fp4", d)
    assert same._desc.format == _lib.BNR_KV_FP4 and same._desc.head_dim == d


@pytest.mark.parametrize("k,scales,error", [
    ((2, 1, 16, 16), None, bitnetrs_amd.InvalidShape),
    ((2, 1, 16, 16), ((2, 1, 16), torch.uint8), bitnetrs_amd.InvalidShape),
    ((2, 1, 16, 17), ((2, 1, 16, 1), torch.uint8), bitnetrs_amd.InvalidShape),
    ((2, 1, 16, 16), ((2, 1, 16, 1), torch.float32), bitnetrs_amd.InvalidShape),
])
def test_pool_refusals(k, scales, error):
    x = torch.zeros(k, dtype=torch.uint8)
    s = [] if scales is None else [torch.zeros(scales[0], dtype=scales[1])] * 2
    with pytest.raises(error):
        bitnetrs_amd.PagedKV.from_tensors(x, x, *s)
    with pytest.raises(bitnetrs_amd.InvalidConfig):
        bitnetrs_amd.PagedKV(1, 16, 1, 33, "fp4", device="cpu")


def test_definition():
    """A code is within half a step of its value, or within 1 of it at the top;
    powers of two, zeros and tiny groups need no case of their own."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((200, 96)) * np.exp(rng.standard_normal((200, 1)) * 20)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-30)
    x[2, :32] = 7 - 2.0 ** -21  # the largest that is cut
    x[3, :32] = 7
    x[4, 40] = np.inf
    x[5, 70] = np.nan
    x[6] = np.float32(3.4028235e38)
    codes, exps = encode(x)
    got = values(codes, exps)
    assert np.array_equal(got[0], np.zeros(96)) and (exps[0] == 25).all()
    assert got[2, 0] == 6 and got[3, 0] == 8 and got[6, 0] == np.float32(6 * 2.0 ** 125)
    assert np.isnan(got[4, 32:64]).all() and np.isfinite(got[4, :32]).all() and np.isfinite(got[4, 64:]).all()
    assert np.isnan(got[5, 64:]).all() and np.isfinite(got[5, :64]).all()
    ok = np.ones(200, bool)
    ok[4:7] = False
    unit = np.repeat(2.0 ** (exps[ok].astype(np.float64) - 127), 32, -1)
    a = np.abs(x[ok].astype(np.float64)) / unit
    step = np.where(a <= 2, 0.5, np.where(a <= 4, 1, 2))
    assert (np.abs(x[ok].astype(np.float64) - got[ok]) / unit <= np.where(a > 6, 1, step / 2)).all()
    m = np.abs(x[ok].reshape(-1, 3, 32)).max(-1)
    assert (np.maximum(m, TINY) / 2.0 ** (exps[ok].astype(np.float64) - 127) < 7).all()
    # ties go to the even code
    tie = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6]] * 4, np.float32).reshape(1, 32)
    assert np.array_equal(values(*encode(tie))[0, :8], [0, 1, 1, 2, 2, 4, 4, 6])
    assert np.array_equal(values(*encode(-tie))[0, :8], [0, -1, -1, -2, -2, -4, -4, -6])
    assert np.array_equal(np.sort(np.unique(E2M1)), E2M1)
