"""dev_rope and rope_scaled_table on the GPU against the rotation in 64 bits."""
import numpy as np
import pytest
import torch

from bitnetrs_amd import InvalidShape, Rope
from fp4_common import Pool4, i32, same

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def rotated(x, positions, rope):
    """In 64 bits, and for each element |x_a| + |x_b| of its pair."""
    y, size, n = x.copy(), np.zeros_like(x), rope.dim // 2
    a = np.arange(n) if rope.layout == "half" else 2 * np.arange(n)
    b = a + n if rope.layout == "half" else a + 1
    angle = (positions.astype(np.float64)[:, None] * rope.rates)[:, None]
    c, s = rope.magnitude * np.cos(angle), rope.magnitude * np.sin(angle)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = abs(rope.magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


def check(got, x, positions, rope, kind):
    """An angle is off by half a place of fp32 at a quarter of a half turn (pi 2^-27), its
    sine and cosine by at most 4 places (2^-22), and four roundings follow
    (magnitude, product, sum: 2^-24 each of the pair's size): under 2^-21 of it.
    The fp64 product of position and rate is off by 2^-52 of itself, as is the
    oracle's.  Then half a step of the type, and half of its least step."""
    want, size = rotated(x, positions, rope)
    turns = np.abs(positions.astype(np.float64))[:, None, None] * np.abs(rope.rates).max()
    bound = size * (2.0 ** -21 + turns * 2.0 ** -50)
    if kind != "f32":
        bound = bound + (np.abs(want) + bound) * torch.finfo(TYPES[kind]).eps / 2 + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all(), float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)))


SHAPES = [(20, 5, 128, 128), (32, 8, 128, 32), (14, 2, 80, 40), (4, 4, 64, 16), (2, 1, 256, 256), (3, 3, 96, 6), (1, 1, 2, 2),
          (5, 1, 34, 34), (2, 2, 512, 512), (3, 1, 130, 128), (2, 1, 7, 6), (4, 2, 48, 24),
          (2, 1, 14, 12)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hq,hkv,d,dim", SHAPES)
def test_rope(backend, kind, layout, hq, hkv, d, dim):
    """Slices of a fused projection's output into tensors of their own; far
    positions; a token that is left out; the elements behind dim as they are."""
    say(f"rope {kind} {layout} {hq}/{hkv}/{d} dim {dim}")
    rng = np.random.default_rng([hq, d, dim])
    n = 33
    rope = Rope(dim, 500000.0, layout=layout, scaling="linear", factor=3.0, magnitude=1.125)
    positions = rng.integers(0, 1 << 20, n)
    positions[:4] = 0, 1, (1 << 31) - 1, 4095
    positions[7] = -1
    x = torch.from_numpy(rng.standard_normal((n, (hq + 2 * hkv) * d)).astype(np.float32)).to(TYPES[kind]).cuda()
    keep = x.clone()
    q, k = x[:, :hq * d].view(n, hq, d), x[:, hq * d:(hq + hkv) * d].view(n, hkv, d)
    outs = [torch.full((n, h, d), 7.0, dtype=x.dtype, device="cuda") for h in (hq, hkv)]
    backend.dev_rope(rope, q, k, i32(positions), *outs)
    assert torch.equal(x, keep)
    for t, o in zip((q, k), outs):
        t, o = t.double().cpu().numpy(), o.double().cpu().numpy()
        assert (o[7] == 7).all()
        on = np.arange(n) != 7
        assert np.array_equal(o[on][..., dim:], t[on][..., dim:])
        check(o[on], t[on], positions[on], rope, kind)
    # in place gives the same bits, and touches nothing else of the projection
    backend.dev_rope(rope, q, k, i32(positions))
    on = torch.arange(n, device="cuda") != 7
    assert torch.equal(q[on], outs[0][on]) and torch.equal(k[on], outs[1][on])
    assert torch.equal(x[7], keep[7]) and torch.equal(x[:, (hq + hkv) * d:], keep[:, (hq + hkv) * d:])


@pytest.mark.parametrize("n", [1, 2, 2047, 2048, 5000])
@pytest.mark.parametrize("dim", [128, 32, 6])
def test_rope_many_tokens(backend, n, dim):
    """One token a workgroup and several of them; heads before tokens; q alone, k alone."""
    say(f"rope {n} tokens dim {dim}")
    rng = np.random.default_rng([n, dim])
    rope = Rope(dim, 10000.0, scaling="parts", factor=8.0, original=512)
    positions = rng.integers(0, 1 << 17, n)
    x = torch.from_numpy(rng.standard_normal((3, n, 128)).astype(np.float32)).cuda()
    q = x.transpose(0, 1)  # [n, 3, 128], a head's tokens side by side
    out = torch.zeros(n, 3, 128, device="cuda")
    backend.dev_rope(rope, q, None, i32(positions), out)
    check(out.double().cpu().numpy(), q.double().cpu().numpy(), positions, rope, "f32")
    back = torch.zeros(3, n, 128, device="cuda").transpose(0, 1)
    backend.dev_rope(rope, None, q, i32(positions), None, back)
    assert torch.equal(back, out)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_alignments(backend, kind, layout):
    """Rows that start at any element have the bits of aligned ones, and what lies
    around them stays."""
    rope, n = Rope(48, 10000.0, layout=layout), 9
    p = i32(np.arange(n) * 77)
    x = torch.randn(n, 3, 64, device="cuda").to(TYPES[kind])
    want = torch.empty_like(x)
    backend.dev_rope(rope, x, None, p, want)
    for first, far in ((1, 64), (2, 64), (4, 64), (8, 64), (0, 65), (0, 66), (0, 68), (0, 72), (4, 68), (2, 72)):
        whole = torch.full((n * 3 * far + 8,), 7.0, dtype=TYPES[kind], device="cuda")
        rows = whole.as_strided((n, 3, 64), (3 * far, far, 1), first)
        out = whole.clone().as_strided((n, 3, 64), (3 * far, far, 1), first)
        rows.copy_(x)
        backend.dev_rope(rope, rows, x, p, out, torch.empty_like(x))
        assert torch.equal(out, want), (first, far)
        backend.dev_rope(rope, rows, None, p)
        assert torch.equal(rows, want), (first, far)
        rows.fill_(7.0)
        assert (whole == 7).all(), (first, far)


def test_shared_rows_as_input(backend):
    """One row for all heads (a stride of zero) may be read, not written."""
    rope = Rope(64, 10000.0)
    x = torch.randn(5, 1, 64, device="cuda").expand(5, 4, 64)
    out = torch.empty(5, 4, 64, device="cuda")
    p = i32([0, 3, 9, 100, 77])
    backend.dev_rope(rope, x, None, p, out)
    assert all(torch.equal(out[:, 0], out[:, h]) for h in range(4))
    check(out.double().cpu().numpy(), x.double().cpu().numpy(), p.cpu().numpy(), rope, "f32")
    with pytest.raises(InvalidShape):
        backend.dev_rope(rope, x, None, p)


@pytest.mark.parametrize("dim", [128, 64, 34])
def test_tables_are_the_same_rotation(backend, dim):
    """dev_paged_append with rope_scaled_table's tables has dev_rope's bits; the
    tables are within the same bound of 64 bits; and a window of them is a part."""
    rng = np.random.default_rng(dim)
    rope = Rope(dim, 500000.0, scaling="ntk", factor=4.0, magnitude=0.75)
    n, hq = 9000, 3
    cos, sin = backend.rope_scaled_table(rope, n)
    angle = np.arange(n)[:, None] * rope.rates
    for t, f in ((cos, np.cos), (sin, np.sin)):
        assert (np.abs(t.cpu().numpy() - 0.75 * f(angle)) <= 2.0 ** -21 + n * 2.0 ** -50).all()
    pos = np.array([0, 1, 4095, 8999, 77])
    q = torch.from_numpy(rng.standard_normal((5, hq, dim)).astype(np.float32)).cuda()
    pool = Pool4(rng, [n] * 5, 1, dim, 16, spread=0.0)
    a, b = torch.empty_like(q), torch.empty_like(q)
    kv = torch.randn(5, 1, dim, device="cuda")
    backend.dev_paged_append(pool.device(), q, kv, kv, a, i32(pos), i32(pool.table), cos, sin)
    backend.dev_rope(rope, q, None, i32(pos), b)
    assert same(a.cpu(), b.cpu())
    some = backend.rope_scaled_table(rope, 100, first=8000)
    assert torch.equal(some[0], cos[8000:8100]) and torch.equal(some[1], sin[8000:8100])


def test_tokens_past_32_bits(backend):
    """Tokens further apart than 32 bits count elements, read and written."""
    rope, far = Rope(64, 10000.0), (1 << 31) + 16
    x = torch.randn(2, 3, 64, device="cuda", dtype=torch.float16)
    big = torch.empty(far + 192, dtype=torch.float16, device="cuda").as_strided((2, 3, 64), (far, 64, 1))
    big.copy_(x)
    p, want, out = i32([7, 123456]), torch.empty_like(x), torch.empty_like(x)
    backend.dev_rope(rope, x, None, p, want)
    backend.dev_rope(rope, big, None, p, out)
    assert torch.equal(out, want)
    backend.dev_rope(rope, big, None, p)
    assert torch.equal(big, want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_more_tokens_than_a_launch_holds(backend, layout):
    """2^26 workgroups' tokens and some: as calls over parts of them."""
    rope, n = Rope(2, 10000.0, layout=layout), (5 << 24) + 5
    x = torch.randn(1 << 20, 1, 2, device="cuda", dtype=torch.bfloat16).repeat(81, 1, 1)[:n].contiguous()
    p = torch.arange(n, dtype=torch.int32, device="cuda")
    p[::7] = -1
    q, k = x.clone(), torch.zeros_like(x)
    backend.dev_rope(rope, q, x, p, None, k)
    for a in range(0, n, 1 << 22):
        b = min(n, a + (1 << 22))
        part = x[a:b].clone()
        backend.dev_rope(rope, part, None, p[a:b])
        assert torch.equal(q[a:b], part)
        part[p[a:b] < 0] = 0
        assert torch.equal(k[a:b], part)


def test_special_values(backend):
    """Infinities and NaN stay in their pairs; zeros stay zero."""
    rope = Rope(8, 100.0)
    x = torch.ones(1, 1, 12, device="cuda")
    x[0, 0, 1], x[0, 0, 6], x[0, 0, 3], x[0, 0, 7], x[0, 0, 9] = np.inf, np.nan, 0, 0, np.nan
    out = torch.empty_like(x)
    backend.dev_rope(rope, x, None, i32([5]), out)
    o = out[0, 0].cpu().numpy()
    assert np.isfinite(o[[0, 4, 8, 10, 11]]).all() and o[3] == 0 and o[7] == 0
    assert np.isnan(o[[2, 6, 9]]).all() and not np.isfinite(o[[1, 5]]).any()


def test_captured(backend):
    """A captured rotation and table follow the positions on each replay."""
    rope = Rope(128, 500000.0, "interleaved")
    q, k = torch.randn(4, 6, 128, device="cuda"), torch.randn(4, 2, 128, device="cuda")
    p = i32([0, 1, 2, 3])
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    tables = backend.rope_scaled_table(rope, 64)
    other = [torch.zeros_like(t) for t in tables]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        backend.dev_rope(rope, q, k, p, qo, ko)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        backend.dev_rope(rope, q, k, p, qo, ko)
        backend.rope_scaled_table(rope, 64, out=other)
    for i in range(4):
        p.copy_(i32(np.arange(4) * 1000 + i))
        q.normal_()
        for t in other:
            t.zero_()
        g.replay()
        want = torch.zeros_like(q), torch.zeros_like(k)
        backend.dev_rope(rope, q, k, p, *want)
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
        assert all(torch.equal(a, b) for a, b in zip(other, tables))


def test_python_refusals(backend):
    rope = Rope(64, 1e4)
    q, p = torch.zeros(3, 2, 64, device="cuda"), i32([0, 1, 2])
    for bad, error in [
        (lambda: backend.dev_rope(rope, None, None, p), TypeError),
        (lambda: backend.dev_rope(rope, q.double(), None, p), TypeError),
        (lambda: backend.dev_rope(rope, q.cpu(), None, p), TypeError),
        (lambda: backend.dev_rope(rope, q, q.half(), p), TypeError),
        (lambda: backend.dev_rope(rope, q, None, p.long()), TypeError),
        (lambda: backend.dev_rope(rope, q, None, p, None, q), TypeError),
        (lambda: backend.dev_rope(rope, q, None, p, q[:, :1].clone()), InvalidShape),
        (lambda: backend.dev_rope(rope, q[0], None, p), InvalidShape),
        (lambda: backend.dev_rope(rope, q[:2], None, p), InvalidShape),
        (lambda: backend.dev_rope(rope, q.transpose(1, 2), None, p), (InvalidShape, TypeError)),
        (lambda: backend.dev_rope(rope, q[..., :32], None, p), InvalidShape),
        (lambda: backend.rope_scaled_table(rope, 4, out=(q[0], q[1])), InvalidShape),
    ]:
        with pytest.raises(error):
            bad()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_operands_of_one_buffer(backend, layout):
    """Slices of fused projections, whose ranges overlap but not their rows, as
    calls on tensors of their own; one tensor as both operands is refused."""
    rope, n, p = Rope(64, 10000.0, layout), 33, i32(np.arange(33) * 7)
    for shape, q_of, k_of in (((n, 12, 64), lambda x: x[:, :8], lambda x: x[:, 8:10]),
                              ((n, 4, 3, 64), lambda x: x[:, :, 0], lambda x: x[:, :, 1]),
                              ((2, 3, n, 64), lambda x: x[0].transpose(0, 1), lambda x: x[1, :2].transpose(0, 1))):
        x = torch.randn(shape, device="cuda", dtype=torch.bfloat16)
        want = x.clone()
        for of in (q_of, k_of):
            part = of(x).contiguous()
            backend.dev_rope(rope, part, None, p)
            of(want).copy_(part)
        backend.dev_rope(rope, q_of(x), k_of(x), p)
        assert torch.equal(x, want)
    q = x[0].transpose(0, 1)
    for k, out in ((q, None), (q[:, 1:], None), (x[1].transpose(0, 1), q)):
        with pytest.raises(InvalidShape):
            backend.dev_rope(rope, q, k, p, None, out)
