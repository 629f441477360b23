"""Paged KV cache without a GPU: what the entry points refuse, before they
touch the device, and what the Python side refuses."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import bitnetrs_amd
from bitnetrs_amd import _lib, backend
from bitnetrs_amd._lib import PagedKVDesc
from common import error_from_parts

# Stands for a context: every refusal comes before the context is used.
CTX = ctypes.create_string_buffer(64)
MEM = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(MEM) + 15) // 16 * 16


def desc(**kw):
    v = dict(k=P, v=P, k_scales=P, v_scales=P, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64,
             format=_lib.BNR_KV_INT8)
    v.update(kw)
    return PagedKVDesc(*[v[n] for n, _ in PagedKVDesc._fields_])


def append(kv, ctx=CTX, **kw):
    a = dict(q=P, k=P, v=P, q_out=P, n_tokens=1, n_heads=4, positions=P, seqs=P, table=P, n_seqs=1,
             stride=2, cos=P, sin=P, n_positions=32)
    a.update(kw)
    return _lib.load().bnr_dev_paged_append(ctx, kv, *a.values(), None)


def read(kv, ctx=CTX, **kw):
    a = dict(table=P, batch=1, stride=2, starts=None, lens=P, k_out=P, v_out=P, cap=8)
    a.update(kw)
    return _lib.load().bnr_dev_paged_read(ctx, kv, *a.values(), None)


def decode(kv, ctx=CTX, **kw):
    a = dict(q=P, n_heads=4, table=P, batch=1, stride=2, lens=P, out=P, workspace=P, bytes=1 << 40)
    a.update(kw)
    return _lib.load().bnr_dev_paged_decode_attention(ctx, kv, *a.values(), None)


def workspace(kv, ctx=CTX, batch=1, n_heads=4, out=True):
    n = ctypes.c_size_t()
    st = _lib.load().bnr_paged_decode_workspace(ctx, kv, batch, n_heads,
                                                ctypes.byref(n) if out else None)
    return st, n.value


BAD_POOLS = [
    (dict(format=4), _lib.BNR_INVALID_CONFIG, "format 4"),
    (dict(format=-1), _lib.BNR_INVALID_CONFIG, "format -1"),
    (dict(n_kv_heads=0), _lib.BNR_INVALID_CONFIG, "n_kv_heads"),
    (dict(n_kv_heads=1 << 20), _lib.BNR_INVALID_CONFIG, "n_kv_heads"),
    (dict(head_dim=0), _lib.BNR_INVALID_SHAPE, "head_dim"),
    (dict(head_dim=63), _lib.BNR_INVALID_CONFIG, "head_dim"),
    (dict(head_dim=514), _lib.BNR_INVALID_CONFIG, "head_dim"),
    (dict(n_pages=0), _lib.BNR_INVALID_SHAPE, "n_pages"),
    (dict(n_pages=1 << 31), _lib.BNR_INVALID_SHAPE, "n_pages"),
    (dict(page_size=0), _lib.BNR_INVALID_SHAPE, "page_size"),
    (dict(page_size=1 << 30), _lib.BNR_INVALID_SHAPE, "table_stride"),
    (dict(n_pages=(1 << 31) - 1, page_size=1 << 29, n_kv_heads=65536), _lib.BNR_INVALID_SHAPE, "2^60"),
    (dict(k=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(v=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(k_scales=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(format=_lib.BNR_KV_FP8, v_scales=None), _lib.BNR_BACKEND_ERROR, "NULL"),
    (dict(format=_lib.BNR_KV_BF16, k=P + 1), _lib.BNR_INVALID_SHAPE, "aligned"),
    (dict(format=_lib.BNR_KV_F32, v=P + 2), _lib.BNR_INVALID_SHAPE, "aligned"),
    (dict(k_scales=P + 2), _lib.BNR_INVALID_SHAPE, "aligned"),
]


@pytest.mark.parametrize("bad,kind,text", BAD_POOLS)
@pytest.mark.parametrize("call", [append, read, decode])
def test_bad_pool_is_refused(call, bad, kind, text):
    assert call(desc(**bad)) == kind
    got, message = error_from_parts()
    assert got == kind and text in message


@pytest.mark.parametrize("call", [append, read, decode])
def test_null_context_and_pool(call):
    assert call(desc(), ctx=None) == _lib.BNR_BACKEND_ERROR
    assert call(None) == _lib.BNR_BACKEND_ERROR


@pytest.mark.parametrize("call,bad,kind", [
    (append, dict(stride=0), _lib.BNR_INVALID_SHAPE),
    (append, dict(stride=(1 << 26) + 1), _lib.BNR_INVALID_SHAPE),
    (append, dict(n_heads=3), _lib.BNR_INVALID_CONFIG),
    (append, dict(n_heads=0), _lib.BNR_INVALID_CONFIG),
    (append, dict(n_heads=1 << 20), _lib.BNR_INVALID_CONFIG),
    (append, dict(n_tokens=1 << 31), _lib.BNR_INVALID_SHAPE),
    (append, dict(n_seqs=1 << 31), _lib.BNR_INVALID_SHAPE),
    (append, dict(seqs=None, n_tokens=2), _lib.BNR_INVALID_SHAPE),
    (append, dict(q=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(q_out=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(k=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(v=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(positions=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(table=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(cos=None), _lib.BNR_BACKEND_ERROR),
    (append, dict(sin=None), _lib.BNR_BACKEND_ERROR),
    (read, dict(stride=0), _lib.BNR_INVALID_SHAPE),
    (read, dict(batch=1 << 31), _lib.BNR_INVALID_SHAPE),
    (read, dict(batch=(1 << 20) + 1), _lib.BNR_INVALID_SHAPE),
    (decode, dict(batch=(1 << 20) + 1), _lib.BNR_INVALID_SHAPE),
    (read, dict(cap=(1 << 30) + 1), _lib.BNR_INVALID_SHAPE),
    (read, dict(cap=1 << 30, batch=(1 << 31) - 1), _lib.BNR_INVALID_SHAPE),
    (read, dict(table=None), _lib.BNR_BACKEND_ERROR),
    (read, dict(lens=None), _lib.BNR_BACKEND_ERROR),
    (read, dict(k_out=None), _lib.BNR_BACKEND_ERROR),
    (read, dict(v_out=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(stride=0), _lib.BNR_INVALID_SHAPE),
    (decode, dict(n_heads=3), _lib.BNR_INVALID_CONFIG),
    (decode, dict(n_heads=0), _lib.BNR_INVALID_CONFIG),
    (decode, dict(batch=1 << 30), _lib.BNR_INVALID_SHAPE),
    (decode, dict(q=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(table=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(lens=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(out=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(workspace=None), _lib.BNR_BACKEND_ERROR),
    (decode, dict(workspace=P + 4), _lib.BNR_INVALID_SHAPE),
    (decode, dict(bytes=4096), _lib.BNR_INVALID_SHAPE),
])
def test_bad_arguments_are_refused(call, bad, kind):
    assert call(desc(), **bad) == kind
    assert error_from_parts()[0] == kind


def test_nothing_to_do_is_no_error():
    # no token, no sequence, no room: nothing is launched
    assert append(desc(), n_tokens=0, k=None) == 0
    assert read(desc(), batch=0, lens=None) == 0
    assert read(desc(), cap=0, k_out=None) == 0
    assert decode(desc(), batch=0, q=None) == 0


def test_workspace_bytes():
    st, n = workspace(desc())
    assert st == 0 and n > 0 and n % 16 == 0
    # one byte less is refused, for the same sizes
    assert decode(desc(), bytes=n - 1) == _lib.BNR_INVALID_SHAPE
    assert workspace(desc(), batch=1000)[1] == n  # batches and kv heads share one
    assert workspace(desc(), n_heads=64)[1] > n
    assert workspace(desc(), n_heads=3)[0] == _lib.BNR_INVALID_CONFIG
    assert workspace(desc(), out=False)[0] == _lib.BNR_BACKEND_ERROR
    assert workspace(None)[0] == _lib.BNR_BACKEND_ERROR


def test_rope_table_refusals():
    f = _lib.load().bnr_dev_rope_table
    assert f(None, 4, 8, 1e4, P, P, None) == _lib.BNR_BACKEND_ERROR
    assert f(CTX, 4, 7, 1e4, P, P, None) == _lib.BNR_INVALID_CONFIG
    assert f(CTX, 4, 8, 0.0, P, P, None) == _lib.BNR_INVALID_CONFIG
    assert f(CTX, (1 << 30) + 1, 8, 1e4, P, P, None) == _lib.BNR_INVALID_SHAPE
    assert f(CTX, 1 << 20, 1 << 20, 1e4, P, P, None) == _lib.BNR_INVALID_SHAPE
    assert f(CTX, 4, 8, 1e4, None, P, None) == _lib.BNR_BACKEND_ERROR
    assert f(CTX, 0, 8, 1e4, None, None, None) == 0


def test_paged_kv_from_tensors():
    kv = bitnetrs_amd.PagedKV(3, 16, 5, 128, "int8", device="cpu")
    assert (kv.fmt, kv.n_pages, kv.page_size, kv.n_kv_heads, kv.head_dim) == ("int8", 3, 16, 5, 128)
    assert kv.k.shape == (3, 5, 16, 128) and kv.k_scales.shape == (3, 5, 16)
    for fmt, dtype in (("f32", torch.float32), ("bf16", torch.bfloat16),
                       ("fp8", torch.float8_e4m3fn), ("int8", torch.int8)):
        assert bitnetrs_amd.PagedKV(1, 16, 1, 8, fmt, device="cpu").k.dtype == dtype
    same = bitnetrs_amd.PagedKV.from_tensors(kv.k, kv.v, kv.k_scales, kv.v_scales)
    assert same.fmt == "int8" and same.k is kv.k
    with pytest.raises(TypeError):  # a pool on the CPU
        kv.desc(0)


@pytest.mark.parametrize("make,error", [
    (lambda z: ((z(2, 1, 16, 8).half(),) * 2, ()), bitnetrs_amd.InvalidConfig),
    (lambda z: ((z(2, 1, 16, 8), z(2, 1, 16, 8).bfloat16()), ()), bitnetrs_amd.InvalidConfig),
    (lambda z: ((z(2, 1, 16, 8), z(2, 1, 8, 8)), ()), bitnetrs_amd.InvalidShape),
    (lambda z: ((z(2, 16, 8),) * 2, ()), bitnetrs_amd.InvalidShape),
    (lambda z: ((z(2, 1, 16, 8),) * 2, (z(2, 1, 16),) * 2), bitnetrs_amd.InvalidConfig),
    (lambda z: ((z(2, 1, 16, 8).char(),) * 2, ()), bitnetrs_amd.InvalidShape),
    (lambda z: ((z(2, 1, 16, 8).char(),) * 2, (z(2, 1, 8),) * 2), bitnetrs_amd.InvalidShape),
    (lambda z: ((z(2, 1, 16, 8).char(),) * 2, (z(2, 1, 16).double(),) * 2), bitnetrs_amd.InvalidShape),
    (lambda z: ((z(2, 1, 8, 16).transpose(2, 3),) * 2, ()), TypeError),
])
def test_paged_kv_refusals(make, error):
    (k, v), scales = make(torch.zeros)
    with pytest.raises(error):
        bitnetrs_amd.PagedKV.from_tensors(k, v, *scales)


def test_unknown_format_name():
    with pytest.raises(bitnetrs_amd.InvalidConfig):
        bitnetrs_amd.PagedKV(1, 16, 1, 8, "int4", device="cpu")


@pytest.mark.parametrize("t,dtype,shape,error", [
    (None, torch.float32, (2,), TypeError), (np.zeros(2, np.float32), torch.float32, (2,), TypeError),
    (torch.zeros(2), torch.float32, (2,), TypeError), ([0.0], torch.float32, (1,), TypeError),
])
def test_operand_check(t, dtype, shape, error):
    # nothing here is a tensor on GPU 0
    with pytest.raises(error):
        backend._on(t, "x", dtype, 0, shape)


def test_operand_sizes():
    backend._check_sizes((torch.zeros(2, 3), "x", 2), (torch.zeros(1), "y", 1))
    with pytest.raises(bitnetrs_amd.InvalidShape):
        backend._check_sizes((torch.zeros(2, 3), "x", 2), (torch.zeros(2), "y", 2))
    with pytest.raises(TypeError):
        backend._check_sizes((None, "x", 2))


def test_format_definitions():
    """The definitions the GPU tests compare with: a code is within half a step
    of its value, the largest value gets the top code, zeros and tiny rows
    need no case of their own."""
    from paged_common import TOP, encode, values

    rng = np.random.default_rng(1)
    x = (rng.standard_normal((40, 64)) * np.exp(rng.standard_normal((40, 1)) * 20)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-30)
    m = np.abs(x).max(-1, keepdims=True)
    for fmt, half in (("int8", 0.5 / 127), ("fp8", 2.0 ** -4)):
        codes, scales = encode(x, fmt)
        back = values(codes, scales)
        # int8: half a step of the row's scale; e4m3: half a step of the value, or of the least one
        room = half * (m if fmt == "int8" else np.maximum(np.abs(x), m * 2.0 ** -6 / 448))
        assert (np.abs(back[2:] - x[2:]) <= room[2:] * (1 + 1e-5)).all()
        assert (back[0] == 0).all()
        top = np.abs(codes.float().numpy()).max(-1)
        assert (top[2:] == TOP[fmt]).all()


def test_index_code_on_the_host():
    """The kernels' own index code: rows stay inside the pool whatever tables,
    positions and sequences hold; shares of a launch cover its work once."""
    native = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
    check = os.path.join(native, "paged_index_check")
    if not os.path.exists(check):
        subprocess.run(["make", "-s", "-C", native, check], check=True)
    out = subprocess.run([check], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


def test_workspace_of_pieces_of_one_head():
    """Shapes that only the kernel of one query head a piece can take ask for no more
    than it uses; none of an accepted shape is out of reach."""
    one = {d: workspace(desc(n_kv_heads=1, head_dim=d), n_heads=1)[1] for d in (26, 64, 130, 512)}
    for kw in (dict(head_dim=512), dict(head_dim=130), dict(head_dim=26), dict(head_dim=64, page_size=8)):
        for n_heads in (2, 16, 64, 65536):
            st, n = workspace(desc(n_kv_heads=1, **kw), n_heads=n_heads)
            assert st == 0 and n == one[kw["head_dim"]], (kw, n_heads, n)
            assert decode(desc(n_kv_heads=1, **kw), n_heads=n_heads, bytes=n - 1) == _lib.BNR_INVALID_SHAPE
    sizes = [workspace(desc(n_kv_heads=1, head_dim=256), n_heads=h)[1] for h in (1, 4, 16, 17, 64, 65536)]
    assert sizes == sorted(sizes) and sizes[-1] <= 36 << 20  # one for many heads serves fewer


@pytest.mark.parametrize("name", ["k", "v", "k_scales", "v_scales", "n_pages", "n_kv_heads", "page_size", "head_dim", "fmt"])
def test_paged_kv_stays_as_it_was_made(name):
    """Calls take a pool by its descriptor, checks by its attributes: neither moves."""
    kv = bitnetrs_amd.PagedKV(3, 16, 2, 64, "int8", device="cpu")
    was = getattr(kv, name)
    with pytest.raises(AttributeError, match=name):
        setattr(kv, name, was.clone() if isinstance(was, torch.Tensor) else was)
    assert getattr(kv, name) is was
    kv.k.fill_(3)  # contents are the caller's
    assert kv._desc.k == kv.k.data_ptr()
