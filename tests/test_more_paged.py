"""Page tables, copies, beam search and rotary forms without a GPU: what the
entry points refuse before they touch the device, and the rotations' rates."""
import ctypes
import math
import re

import numpy as np
import pytest

import bitnetrs_amd
from bitnetrs_amd import _lib, Rope
from bitnetrs_amd._lib import HeadsDesc, RopeDesc
from common import error_from_parts
from test_paged import CTX, desc

# separate places for separate operands; nothing is read before a refusal
MEM = ctypes.create_string_buffer(1 << 20)
BASE = (ctypes.addressof(MEM) + 4095) // 4096 * 4096


def at(i):
    return BASE + 8192 * i


def extend(ctx=CTX, **kw):
    a = dict(table=at(0), n_seqs=3, stride=4, page=16, lens=at(1), new=at(2), free=at(3), cap=10, count=at(4), seqs=at(5),
             positions=at(6), slots=at(7), n_tokens=20, offsets=at(8), lens_out=at(9), count_out=at(10))
    a.update(kw)
    return _lib.load().bnr_dev_paged_extend(ctx, *a.values(), None)


def release(ctx=CTX, **kw):
    a = dict(table=at(0), n_seqs=3, stride=4, page=16, lens=at(1), which=at(2), keep=at(3), free=at(4), cap=10, count=at(5),
             lens_out=at(6), count_out=at(7))
    a.update(kw)
    return _lib.load().bnr_dev_paged_release(ctx, *a.values(), None)


def copy(kv=None, ctx=CTX, **kw):
    a = dict(table=at(0), n_seqs=3, stride=2, src=at(1), starts=at(2), lens=at(3))
    a.update(kw)
    return _lib.load().bnr_dev_paged_copy(ctx, desc() if kv is None else kv, *a.values(), None)


def select(ctx=CTX, **kw):
    a = dict(logits=at(0), stride=100, batch=2, beams=4, vocab=100, k=4, scores=at(1), done=at(2), eos=5, tokens=at(3),
             parents=at(4), scores_out=at(5), done_out=at(6), workspace=at(7), bytes=1 << 14)
    a.update(kw)
    return _lib.load().bnr_dev_beam_select(ctx, *a.values(), None)


def reorder(ctx=CTX, **kw):
    a = dict(table=at(0), batch=2, beams=4, stride=10, parents=at(1), out=at(2), src=at(3))
    a.update(kw)
    return _lib.load().bnr_dev_beam_reorder(ctx, *a.values(), None)


RATES = (ctypes.c_double * 256)(*[0.5] * 256)


def rotation(rates=RATES, n=32, layout=0, magnitude=1.0):
    d = RopeDesc(ctypes.addressof(rates) if rates is not None else None, n, layout, magnitude)
    d.kept = rates  # the descriptor has only their address
    return d


def heads(i=1, o=None, n=4, it=256, ih=64, ot=256, oh=64):
    return bytes(HeadsDesc(at(i), at(i) if o is None else o, n, it, ih, ot, oh))


def rope(ctx=CTX, r=None, **kw):
    a = dict(type=0, n=4, d=64, positions=at(0), q=heads(1), k=heads(3))
    a.update(kw)
    return _lib.load().bnr_dev_rope(ctx, rotation() if r is None else r, *a.values(), None)


def table(ctx=CTX, r=None, **kw):
    a = dict(first=0, n=8, cos=at(0), sin=at(1))
    a.update(kw)
    return _lib.load().bnr_dev_rope_scaled_table(ctx, rotation() if r is None else r, *a.values(), None)


SHAPE, CONFIG, BACKEND = _lib.BNR_INVALID_SHAPE, _lib.BNR_INVALID_CONFIG, _lib.BNR_BACKEND_ERROR

REFUSED = [
    (extend, dict(n_seqs=4097), SHAPE, "n_seqs"),
    (extend, dict(page=0), SHAPE, "page_size"),
    (extend, dict(stride=0), SHAPE, "table_stride"),
    (extend, dict(stride=1 << 26, page=32), SHAPE, "table_stride"),
    (extend, dict(cap=1 << 31), SHAPE, "free_cap"),
    (extend, dict(n_tokens=1 << 31), SHAPE, "n_tokens"),
    *[(extend, {n: None}, BACKEND, "NULL") for n in
      ("table", "lens", "new", "free", "count", "seqs", "positions", "offsets", "lens_out", "count_out")],
    (extend, dict(lens_out=at(1)), SHAPE, "lens_out and lens"),
    (extend, dict(count_out=at(4)), SHAPE, "free_count_out and free_count"),
    (extend, dict(seqs=at(6) + 76), SHAPE, "seqs and positions"),
    (extend, dict(slots=at(8) - 8), SHAPE, "slots and offsets"),
    (extend, dict(lens=at(0) + 44), SHAPE, "block_table and lens"),
    (release, dict(n_seqs=4097), SHAPE, "n_seqs"),
    (release, dict(page=1 << 31), SHAPE, "page_size"),
    *[(release, {n: None}, BACKEND, "NULL") for n in ("table", "lens", "which", "free", "count", "lens_out", "count_out")],
    (release, dict(lens_out=at(1)), SHAPE, "lens_out and lens"),
    (release, dict(count_out=at(5)), SHAPE, "free_count_out and free_count"),
    (release, dict(free=at(0) + 4), SHAPE, "block_table and free_pages"),
    (copy, dict(stride=0), SHAPE, "table_stride"),
    (copy, dict(n_seqs=(1 << 20) + 1), SHAPE, "batch"),
    *[(copy, {n: None}, BACKEND, "NULL") for n in ("table", "src", "lens")],
    (select, dict(beams=0), CONFIG, "beams"),
    (select, dict(beams=33), CONFIG, "beams"),
    (select, dict(k=0), CONFIG, "continuations"),
    (select, dict(k=33), CONFIG, "continuations"),
    (select, dict(vocab=3, k=4), CONFIG, "continuations"),
    (select, dict(vocab=0), SHAPE, "vocab"),
    (select, dict(vocab=(1 << 30) + 1, stride=1 << 31), SHAPE, "vocab"),
    (select, dict(stride=99), SHAPE, "row_stride"),
    (select, dict(batch=1 << 20), SHAPE, "batch"),
    (select, dict(eos=-1), CONFIG, "eos"),
    (select, dict(eos=100), CONFIG, "eos"),
    (select, dict(eos=-2, done=None), CONFIG, "eos"),
    (select, dict(bytes=16), SHAPE, "workspace"),
    (select, dict(workspace=at(7) + 4), SHAPE, "aligned"),
    *[(select, {n: None}, BACKEND, "NULL") for n in ("logits", "scores", "tokens", "parents", "scores_out", "workspace")],
    (select, dict(scores_out=at(1)), SHAPE, "scores_out and scores"),
    (select, dict(done_out=at(2)), SHAPE, "done_out and done"),
    (select, dict(tokens=at(4)), SHAPE, "tokens and parents"),
    (reorder, dict(beams=0), CONFIG, "beams"),
    (reorder, dict(beams=33), CONFIG, "beams"),
    (reorder, dict(stride=0), SHAPE, "table_stride"),
    (reorder, dict(batch=1 << 20), SHAPE, "batch"),
    *[(reorder, {n: None}, BACKEND, "NULL") for n in ("table", "parents", "out", "src")],
    (reorder, dict(out=at(0)), SHAPE, "table_out and block_table"),
    (reorder, dict(src=at(1)), SHAPE, "src and parents"),
    (rope, dict(r=rotation(n=0)), CONFIG, "pairs"),
    (rope, dict(r=rotation(n=257)), CONFIG, "pairs"),
    (rope, dict(r=rotation(layout=2)), CONFIG, "layout"),
    (rope, dict(r=rotation(magnitude=math.inf)), CONFIG, "magnitude"),
    (rope, dict(r=rotation(rates=None)), BACKEND, "rates"),
    (rope, dict(r=rotation(rates=(ctypes.c_double * 32)(math.nan))), CONFIG, "rate 0"),
    (rope, dict(r=rotation(rates=(ctypes.c_double * 32)(1.0, -1e5))), CONFIG, "rate 1"),
    (rope, dict(type=3), CONFIG, "type"),
    (rope, dict(d=62), SHAPE, "head_dim"),
    (rope, dict(n=1 << 31), SHAPE, "n_tokens"),
    (rope, dict(positions=None), BACKEND, "positions"),
    (rope, dict(q=heads(1, n=1 << 20)), CONFIG, "heads"),
    (rope, dict(q=heads(1, ot=255)), SHAPE, "output rows"),
    (rope, dict(q=heads(1, oh=63)), SHAPE, "output rows"),
    (rope, dict(q=heads(1, ot=0)), SHAPE, "output rows"),
    (rope, dict(k=heads(3, o=at(3) + 4)), SHAPE, "in place"),
    (rope, dict(k=heads(3, it=512)), SHAPE, "in place"),
    (rope, dict(q=heads(1, it=1 << 41, ot=1 << 41)), SHAPE, "strides"),
    (rope, dict(q=bytes(HeadsDesc(None, at(1), 4, 256, 64, 256, 64))), BACKEND, "NULL"),
    (rope, dict(q=bytes(HeadsDesc(at(1) + 2, at(1) + 2, 4, 256, 64, 256, 64))), SHAPE, "aligned"),
    (table, dict(r=rotation(n=0)), CONFIG, "pairs"),
    (table, dict(n=(1 << 30) + 1), SHAPE, "n_positions"),
    (table, dict(first=1 << 31), SHAPE, "first"),
    (table, dict(cos=None), BACKEND, "NULL"),
]


@pytest.mark.parametrize("call,bad,kind,text", REFUSED)
def test_refused(call, bad, kind, text):
    assert call(**bad) == kind
    assert text in error_from_parts()[1]


@pytest.mark.parametrize("call", [extend, release, copy, select, reorder, rope, table])
def test_null_context(call):
    assert call(ctx=None) == BACKEND
    assert "context is NULL" in error_from_parts()[1]


@pytest.mark.parametrize("call,nothing", [
    (copy, dict(n_seqs=0)), (select, dict(batch=0)), (reorder, dict(batch=0)), (rope, dict(n=0)), (table, dict(n=0)),
    (rope, dict(q=None, k=None)), (rope, dict(q=heads(1, n=0), k=None)),
])
def test_nothing_to_do_is_no_error(call, nothing):
    assert call(**nothing) == _lib.BNR_OK


def test_packed_heads_are_the_structure():
    from bitnetrs_amd import backend

    v = [at(1), at(2), 3, 4, 5, 6, (1 << 40) + 7]
    assert backend._pack_heads(*v) == bytes(HeadsDesc(*v))


def test_beam_workspace():
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.bnr_beam_workspace(CTX, 2, 4, 100, 4, ctypes.byref(n)) == _lib.BNR_OK and 0 < n.value <= 1 << 14
    assert lib.bnr_beam_workspace(CTX, 0, 4, 100, 4, ctypes.byref(n)) == _lib.BNR_OK and n.value == 0
    assert lib.bnr_beam_workspace(CTX, 2, 4, 100, 4, None) == BACKEND
    assert lib.bnr_beam_workspace(None, 2, 4, 100, 4, ctypes.byref(n)) == BACKEND
    assert lib.bnr_beam_workspace(CTX, 2, 0, 100, 4, ctypes.byref(n)) == CONFIG


# ---------------------------------------------------------------------------
# rotations
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim,theta", [(2, 1e4), (32, 1e4), (128, 500000.0), (512, 1e6)])
def test_rates(dim, theta):
    r = Rope(dim, theta)
    want = [theta ** (-2 * i / dim) for i in range(dim // 2)]
    assert r.dim == dim and r.magnitude == 1 and np.allclose(r.rates, want, rtol=1e-14, atol=0)
    assert np.allclose(Rope(dim, theta, scaling="linear", factor=4).rates, r.rates / 4, rtol=1e-14, atol=0)
    same = Rope.from_rates(r.rates, "interleaved", 1.5)
    assert np.array_equal(same.rates, r.rates) and (same.layout, same.magnitude) == ("interleaved", 1.5)


def test_scaled_rates():
    plain = Rope(128, 10000.0).rates
    ntk = Rope(128, 10000.0, scaling="ntk", factor=8).rates
    assert ntk[0] == 1 and abs(ntk[-1] * 8 / plain[-1] - 1) < 1e-12  # the slowest pair is stretched by the factor
    assert (np.diff(ntk / plain) < 0).all()
    parts = Rope(128, 10000.0, scaling="parts", factor=8, original=4096, alpha=1, beta=32, magnitude=1.2)
    turns = 4096 * plain / (2 * math.pi)
    assert np.array_equal(parts.rates[turns >= 32], plain[turns >= 32])
    assert np.allclose(parts.rates[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (parts.rates[mid] < plain[mid]).all() and (parts.rates[mid] > plain[mid] / 8).all()
    i = int(np.nonzero(mid)[0][0])
    g = (turns[i] - 1) / 31
    assert abs(parts.rates[i] / (plain[i] * (g + (1 - g) / 8)) - 1) < 1e-12 and parts.magnitude == 1.2


@pytest.mark.parametrize("bad", [
    dict(dim=0), dict(dim=33), dict(dim=514), dict(dim=2.0), dict(theta=0.0), dict(theta=math.nan), dict(theta=math.inf),
    dict(layout="both"), dict(scaling="other"), dict(scaling="linear", factor=0.0), dict(scaling="linear", factor=math.nan),
    dict(scaling="parts", factor=2.0), dict(scaling="parts", factor=2.0, original=10, alpha=4, beta=4),
    dict(scaling="ntk", factor=2.0, dim=2), dict(magnitude=math.nan),
])
def test_rope_refusals(bad):
    with pytest.raises(bitnetrs_amd.InvalidConfig):
        Rope(**{**dict(dim=64, theta=1e4), **bad})


@pytest.mark.parametrize("rates", [[], [[1.0]], [math.inf], np.ones(257)])
def test_rope_from_rates_refusals(rates):
    with pytest.raises(bitnetrs_amd.InvalidConfig):
        Rope.from_rates(rates)


def test_rope_is_fixed():
    r = Rope(64, 1e4)
    with pytest.raises(AttributeError):
        r.rates = np.ones(32)
    with pytest.raises(ValueError):
        r.rates[0] = 2
    own = np.ones(4)
    kept = Rope.from_rates(own)
    own[:] = 7
    assert (kept.rates == 1).all()


def beam_need(batch, beams, vocab, k):
    """What a selection asks for, from its refusal of a workspace of no bytes."""
    assert select(batch=batch, beams=beams, vocab=vocab, stride=vocab, k=k, bytes=0, eos=0) == SHAPE
    return int(re.search(r"workspace of (\d+) bytes", error_from_parts()[1]).group(1))


@pytest.mark.parametrize("vocab", [40, 2000, 32000, 128256])
def test_beam_workspace_serves_smaller_calls(vocab):
    """A workspace serves every call with no more requests, beams, tokens and
    continuations: a server makes one for its largest."""
    lib, n = _lib.load(), ctypes.c_size_t()

    def room(batch, beams, vocab, k):
        assert lib.bnr_beam_workspace(CTX, batch, beams, vocab, k, ctypes.byref(n)) == _lib.BNR_OK
        return n.value

    batches, ks = [1, 2, 3, 4, 7, 12, 15, 16, 31, 32, 128, 300], [1, 2, 5, 8, 15, 16, 17, 31, 32]
    for beams in (1, 4, 8, 32):
        for k in ks:
            most = 0
            for b in batches:
                most = max(most, beam_need(b, beams, vocab, k))
                assert room(b, beams, vocab, k) >= most, (b, beams, k)
    for beams in (1, 8, 32):
        for b in batches:
            most = 0
            for k in ks:
                most = max(most, beam_need(b, beams, vocab, k))
                assert room(b, beams, vocab, k) >= most, (b, beams, k)
    for b in batches:
        most = 0
        for beams in range(1, 33):
            most = max(most, beam_need(b, beams, vocab, 8), beam_need(b, beams, vocab // 2, 8))
            assert room(b, beams, vocab, 8) >= most, (b, beams)


# ---------------------------------------------------------------------------
# rotations whose operands meet
# ---------------------------------------------------------------------------
def place(base, n_heads, token, head, out=None, out_token=None, out_head=None):
    """Heads at elements of one buffer (fp32); in place unless `out` is given."""
    out, out_token, out_head = (base, token, head) if out is None else (out, out_token, out_head)
    return bytes(HeadsDesc(BASE + 4 * base, BASE + 4 * out, n_heads, token, head, out_token, out_head))


APART = [  # q, k of heads of 64
    (dict(base=0, n_heads=4, token=384, head=64), dict(base=256, n_heads=1, token=384, head=64)),  # a fused projection
    (dict(base=0, n_heads=4, token=512, head=128), dict(base=64, n_heads=4, token=512, head=128)),  # head by head
    (dict(base=0, n_heads=2, token=768, head=192), dict(base=400, n_heads=3, token=768, head=80)),
    (dict(base=0, n_heads=2, token=64, head=1024), dict(base=256, n_heads=2, token=64, head=1024)),  # tokens within heads
]
MEET = [
    (dict(base=0, n_heads=4, token=256, head=64), dict(base=0, n_heads=4, token=256, head=64)),
    (dict(base=0, n_heads=4, token=384, head=64), dict(base=255, n_heads=2, token=384, head=64)),
    (dict(base=0, n_heads=4, token=384, head=64), dict(base=256, n_heads=3, token=384, head=64)),
    (dict(base=0, n_heads=4, token=512, head=128), dict(base=60, n_heads=4, token=512, head=128)),
    (dict(base=0, n_heads=4, token=256, head=64, out=4096, out_token=256, out_head=64),
     dict(base=4100, n_heads=2, token=256, head=64, out=9000, out_token=128, out_head=64)),  # k reads what q writes
    (dict(base=0, n_heads=1, token=128, head=64), dict(base=64, n_heads=1, token=256, head=64)),
]


@pytest.mark.parametrize("q,k", APART)
def test_rope_operands_of_one_buffer(q, k):
    """Accepted: the next refusal is the positions'."""
    for a, b in ((q, k), (k, q)):
        assert rope(q=place(**a), k=place(**b), positions=None) == BACKEND
        assert "positions" in error_from_parts()[1]


@pytest.mark.parametrize("q,k", MEET)
def test_rope_operands_that_meet_are_refused(q, k):
    for a, b in ((q, k), (k, q)):
        assert rope(q=place(**a), k=place(**b)) == SHAPE
        assert "apart" in error_from_parts()[1]


def test_rope_operands_against_their_elements():
    """Random places in one buffer: refused where an element that one operand
    writes is the other's, and nowhere else (operands of equal token distance)."""
    rng = np.random.default_rng(11)
    n, d, seen = 3, 4, [0, 0]
    r = rotation(n=2)
    for _ in range(4000):
        token = int(rng.integers(4, 40))
        sides = []
        for _ in range(2):
            m, head = int(rng.integers(1, 4)), int(rng.integers(4, 40))
            base, away = int(rng.integers(0, 60)), bool(rng.random() < 0.3)
            args = dict(base=base, n_heads=m, token=token, head=head)
            if away:
                args.update(out=base + 400, out_token=token, out_head=head)
            at = {base + i * token + h * head + e for i in range(n) for h in range(m) for e in range(d)}
            sides.append((args, at, {x + 400 for x in at} if away else at))
        if any(len(at) != n * d * a["n_heads"] for a, at, _ in sides):
            continue
        (a, ai, ao), (b, bi, bo) = sides
        kind = rope(r=r, n=n, d=d, positions=None, q=place(**a), k=place(**b))
        text = error_from_parts()[1]
        if "output rows" in text:  # neither heads within tokens nor tokens within heads
            continue
        meet = bool(ao & bo or ao & bi or ai & bo)
        assert (kind == SHAPE and "apart" in text) == meet and (kind == BACKEND) == (not meet), (a, b)
        seen[meet] += 1
    assert min(seen) > 50


@pytest.mark.parametrize("bad", [dict(positions=at(1)), dict(positions=at(3) + 16)])
def test_rope_positions_in_an_output(bad):
    assert rope(**bad) == SHAPE and "positions" in error_from_parts()[1]


@pytest.mark.parametrize("off", [0, 4, 4 * (8 * 32 - 1), -4])
def test_rotation_tables_apart(off):
    assert table(sin=at(0) + off) == SHAPE and "apart" in error_from_parts()[1]


@pytest.mark.filterwarnings("error")
@pytest.mark.parametrize("bad", [
    dict(scaling="ntk", factor=1e308), dict(scaling="ntk", factor=1e300, theta=1e200), dict(theta=1e-300, dim=512, scaling="linear", factor=1e-20),
    dict(scaling="parts", factor=2.0, original=math.nan), dict(scaling="parts", factor=2.0, original=10, alpha=-math.inf),
])
def test_rates_that_are_no_numbers_are_refused(bad):
    with pytest.raises(bitnetrs_amd.InvalidConfig):
        Rope(**{**dict(dim=64, theta=1e4), **bad})
