"""Page tables, copies and beam search on the GPU against their definitions in
numpy (tests/beam_common.py), and a search as a server would run it."""
import numpy as np
import pytest
import torch

from beam_common import extend, pages_of, release, reorder, select
from bitnetrs_amd import InvalidConfig, InvalidShape, PagedKV, Rope
from fp4_common import attention, attention_bound, encode, i32, same, values

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# ---------------------------------------------------------------------------
# extend and release
# ---------------------------------------------------------------------------
class Tables:
    def __init__(self, rng, lens, width, page, n_free, cap=None):
        self.page, self.lens = page, np.array(lens, np.int32)
        have = [pages_of(min(max(n, 0), width * page), page) for n in lens]
        order = rng.permutation(sum(have) + n_free).astype(np.int32)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for s, h in enumerate(have):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.free = np.concatenate([order[at:], np.full((cap or n_free) - n_free, -5, np.int32)])
        self.count = n_free


def run_extend(be, t, new, n_tokens, slots=True, count=None):
    n, count = len(t.lens), t.count if count is None else count
    table, lens, free = cuda(t.table), cuda(t.lens), cuda(t.free)
    seqs, pos, off, lo, co = (torch.full((m,), 99, dtype=torch.int32, device="cuda")
                              for m in (n_tokens, n_tokens, n + 1, n, 1))
    sl = torch.full((n_tokens,), 99, dtype=torch.int64, device="cuda") if slots else None
    be.dev_paged_extend(table, lens, i32(new), free, i32([count]), t.page, seqs, pos, off, lo, co, slots=sl)
    want = extend(t.table, t.lens, new, t.free, count, t.page, n_tokens)
    got = [x.cpu().numpy() for x in (table, lo, co, seqs, pos, off)]
    assert np.array_equal(cuda(t.lens).cpu(), lens.cpu()) and np.array_equal(free.cpu().numpy(), t.free)
    for g, w, name in zip(got, (want[0], want[1], [want[2]], want[3], want[4], want[6]),
                          ("table", "lens", "count", "seqs", "positions", "offsets")):
        assert np.array_equal(g, w), name
    if slots:
        assert np.array_equal(sl.cpu().numpy(), want[5]), "slots"
    return want


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 257, 1000, 4096])
@pytest.mark.parametrize("page", [1, 16, 48])
def test_extend(backend, n, page):
    """A decode step and ragged prompts, sequences without a row or new token."""
    say(f"extend {n} sequences, pages of {page}")
    rng = np.random.default_rng([n, page])
    lens = rng.integers(0, 60, n)
    width = pages_of(160, page) + 1
    t = Tables(rng, lens, width, page, n * width)
    run_extend(backend, t, np.ones(n, np.int32), n)
    new = rng.integers(0, 100, n) * (rng.random(n) < 0.8)
    run_extend(backend, t, new, int(new.sum()))
    run_extend(backend, t, new, int(new.sum()) + 777, slots=False)
    run_extend(backend, t, np.zeros(n, np.int32), 5)


@pytest.mark.parametrize("n", [1, 7, 300, 1025])
def test_extend_runs_out(backend, n):
    """Too few pages, too few places, no room in the table, lengths and counts
    that are none: the same prefix of sequences is served."""
    rng = np.random.default_rng(n)
    page, width = 16, 9
    lens = rng.integers(0, 100, n)
    lens[rng.random(n) < 0.1] = -4
    t = Tables(rng, lens, width, page, 2 * n, cap=2 * n + 3)
    new = rng.integers(-2, 80, n)
    new[rng.random(n) < 0.05] = (1 << 31) - 1
    total = int(np.clip(new, 0, 200).sum())
    for count in (0, 1, n // 2, n, 2 * n, 2 * n + 3, 1 << 30, -3):
        say(f"extend {n}, {count} pages")
        run_extend(backend, t, new, total, count=count)
    for places in (0, 1, total // 3):
        say(f"extend {n}, {places} places")
        run_extend(backend, t, new, places)


def test_extend_no_sequences(backend):
    seqs, pos, off, co = i32([9, 9]), i32([9, 9]), i32([9]), i32([9])
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    backend.dev_paged_extend(none, i32([]), i32([]), i32([4, 5]), i32([2]), 16, seqs, pos, off, i32([]), co)
    assert seqs.tolist() == [-1, -1] and pos.tolist() == [-1, -1] and off.tolist() == [0] and co.tolist() == [2]


@pytest.mark.parametrize("n", [1, 5, 64, 300, 4096])
@pytest.mark.parametrize("with_keep", [False, True])
def test_release(backend, n, with_keep):
    say(f"release {n} sequences")
    rng = np.random.default_rng([n, with_keep])
    page, width = 16, 8
    lens = rng.integers(-2, width * page + 40, n)
    t = Tables(rng, lens, width, page, 10, cap=10 + n * width)
    keep = rng.integers(-1, 5, n).astype(np.int32) if with_keep else None
    which = (rng.random(n) < 0.5).astype(np.uint8) * 255
    for cap in (10, 10 + n, 10 + n * width):
        table, free = cuda(t.table), cuda(t.free[:cap])
        lo, co = i32([99] * n), i32([99])
        backend.dev_paged_release(table, cuda(t.lens), cuda(which), free, i32([10]), page, lo, co,
                                  keep=None if keep is None else cuda(keep))
        want = release(t.table, t.lens, which, keep, t.free[:cap], 10, page)
        for g, w, name in zip((table, lo, free, co), (want[0], want[1], want[2], [want[3]]),
                              ("table", "lens", "free", "count")):
            assert np.array_equal(g.cpu().numpy(), w), (cap, name)


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
def run_select(be, logits, scores, k, done=None, eos=-1, ws=None):
    B, K, V = logits.shape
    tokens, parents = (torch.full((B, k), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    out, ended = torch.full((B, k), 99.0, device="cuda"), torch.full((B, k), 99, dtype=torch.uint8, device="cuda")
    ws = be.beam_workspace(B, K, V, k) if ws is None else ws
    be.dev_beam_select(logits, scores, tokens, parents, out, ws, done=done, eos=eos, done_out=ended)
    return [x.cpu().numpy() for x in (tokens, parents, out, ended)]


def check_select(be, logits, scores, k, done=None, eos=-1, device=None):
    """Tokens, parents and ends equal.  lse: a term exp(d), d = x - max, is off by a
    place of exp2 (2^-23) and by the roundings of d and of its product with
    log2(e) in two (3 |d| 2^-24 together); d's mean under the softmax is at most
    the entropy, ln V < 14, so that is 2^-18.5 of the sum; a thread adds at most
    64 terms (2^-18).  Under 2^-17 in all, and 2^-16 between two beams: the oracle's
    neighbours of different beams are further apart.  A score: that, and half a step
    of fp32."""
    tokens, parents, best, ended, gap = select(logits, scores, k, done, eos)
    assert gap > 2.0 ** -16, "inputs whose order hangs on rounding"
    got = run_select(be, cuda(logits) if device is None else device, cuda(scores), k,
                     None if done is None else cuda(done), eos)
    assert np.array_equal(got[1], parents), "parents"
    assert np.array_equal(got[0], tokens), "tokens"
    assert np.array_equal(got[3], ended), "ends"
    inf = np.isinf(best)
    assert np.array_equal(np.isneginf(got[2]), inf)
    off = np.abs(got[2][~inf] - best[~inf])
    assert (off <= 2.0 ** -17 + np.abs(best[~inf]) * 2.0 ** -24).all()
    return got


@pytest.mark.parametrize("B,K,V,k", [(1, 1, 1, 1), (1, 4, 128256, 4), (3, 2, 5, 2), (2, 3, 1001, 3), (1, 1, 300000, 32),
                                     (5, 4, 4097, 4), (2, 32, 2000, 32), (1, 32, 40, 32), (40, 3, 777, 6), (1, 2, 70001, 5),
                                     (300, 4, 100, 4), (2, 5, 32000, 10), (1, 8, 3, 3)])
def test_select(backend, B, K, V, k):
    say(f"select {B}x{K} vocab {V} k {k}")
    rng = np.random.default_rng([B, K, V])
    logits = (3 * rng.standard_normal((B, K, V))).astype(np.float32)
    scores = (-4 * rng.random((B, K))).astype(np.float32)
    check_select(backend, logits, scores, k)


@pytest.mark.parametrize("V", [100, 1003, 9000, 40000])
def test_select_ended_and_first_step(backend, V):
    """Ended beams go on with the end's token; a first step's beams but one have no score."""
    rng = np.random.default_rng(V)
    B, K = 6, 4
    logits = (2 * rng.standard_normal((B, K, V))).astype(np.float32)
    scores = (-6 * rng.random((B, K))).astype(np.float32)
    done = (rng.random((B, K)) < 0.4).astype(np.uint8) * 2
    done[0] = 1
    done[1] = 0
    for eos in (0, 2, V - 1):
        check_select(backend, logits, scores, K, done, eos)
    check_select(backend, logits, scores, K, None, int(np.argmax(logits[0, 0])))
    scores[:, 1:] = -np.inf
    check_select(backend, logits, scores, K)
    scores[2] = -np.inf
    scores[3, 0] = np.nan
    scores[4, 0] = np.inf
    check_select(backend, logits, scores, K, done, 1)


@pytest.mark.parametrize("V", [64, 5000, 20001])
def test_select_ties_and_masks(backend, V):
    """Equal logits, in whole rows too (more than a tile's list has room for):
    the lowest tokens; masked tokens; rows with one token left or none."""
    B, K, k = 4, 3, 8
    logits = np.zeros((B, K, V), np.float32)
    scores = np.array([[-1, -1.5, -3], [0, -1, -2], [-1, -2, -4], [0, 0, 0]], np.float32)
    logits[1, :, V // 2:] = 1.0
    logits[2] = -np.inf
    logits[2, 0, V - 1], logits[2, 1, 7], logits[2, 1, 40] = 3, 1, 1
    rng = np.random.default_rng(V)
    logits[3] = rng.integers(-2, 3, (K, V))
    check_select(backend, logits, scores, k)
    # the same in lists that were full before: large first logits, then a flood of equal ones
    logits[0, :, :50] = 5 + 0.25 * np.arange(50, dtype=np.float32)
    logits[0, :, 50:] = 30
    logits[1] = np.sort(rng.standard_normal((K, V)).astype(np.float32), -1)
    check_select(backend, logits, scores, k)


@pytest.mark.parametrize("V", [77, 4500])
def test_select_not_finite(backend, V):
    """A NaN or +infinity leaves a beam without a continuation, and no other."""
    rng = np.random.default_rng(V)
    B, K = 4, 4
    logits = (2 * rng.standard_normal((B, K, V))).astype(np.float32)
    scores = (-2 * rng.random((B, K))).astype(np.float32)
    logits[0, 1, V - 1] = np.nan
    logits[1, 2, 3] = np.inf
    logits[2] = np.nan
    logits[3, 0] = -np.inf
    logits[3, 1, 5:] = np.nan
    check_select(backend, logits, scores, K)


def test_select_wide_logits(backend):
    """Logits hundreds apart, large ones, and scores far below zero."""
    rng = np.random.default_rng(8)
    logits = (200 * rng.standard_normal((3, 4, 2500))).astype(np.float32)
    logits[1] += 10000
    scores = (-300 * rng.random((3, 4))).astype(np.float32)
    tokens, parents, best, _, gap = select(logits, scores, 4)
    assert gap > 2.0 ** -10
    got = run_select(backend, cuda(logits), cuda(scores), 4)
    assert np.array_equal(got[0], tokens) and np.array_equal(got[1], parents)
    assert (np.abs(got[2] - best) <= 2.0 ** -16 + np.abs(best) * 2.0 ** -24).all()


@pytest.mark.parametrize("V,pad", [(1000, 24), (1001, 3), (129, 127)])
def test_select_padded_rows(backend, V, pad):
    """Rows further apart than the vocabulary, what lies between them unread."""
    rng = np.random.default_rng(V)
    logits = (2 * rng.standard_normal((3, 4, V))).astype(np.float32)
    wide = torch.full((3, 4, V + pad), float("nan"), device="cuda")
    wide[..., :V] = cuda(logits)
    check_select(backend, logits, (-rng.random((3, 4))).astype(np.float32), 4, device=wide[..., :V])
    one = wide[:1, :1, :V]
    check_select(backend, logits[:1, :1], np.zeros((1, 1), np.float32), 4, device=one)


def test_select_rows_past_32_bits(backend):
    """Rows further apart than 32 bits count elements."""
    rng = np.random.default_rng(3)
    V, far = 2000, (1 << 31) + 8
    logits = (2 * rng.standard_normal((1, 3, V))).astype(np.float32)
    wide = torch.empty(2 * far + V, device="cuda").as_strided((1, 3, V), (3 * far, far, 1))
    wide.copy_(cuda(logits))
    check_select(backend, logits, np.array([[-1, -0.5, -2]], np.float32), 3, device=wide)


def test_select_same_bits_captured(backend):
    """Replayed on new logits; one workspace for two shapes, one after the other."""
    B, K, V = 4, 4, 30001
    x, scores = torch.randn(B, K, V, device="cuda"), torch.zeros(B, K, device="cuda")
    ws = backend.beam_workspace(B, K, V, K)
    tokens, parents = (torch.zeros(B, K, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.zeros(B, K, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        backend.dev_beam_select(x, scores, tokens, parents, out, ws)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        backend.dev_beam_select(x, scores, tokens, parents, out, ws)
    for i in range(4):
        x.normal_().mul_(3)
        scores.uniform_(-3, 0)
        run_select(backend, x[:1, :, :100].contiguous(), scores[:1], 2, ws=ws)
        g.replay()
        want = run_select(backend, x, scores, K)
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(parents.cpu().numpy(), want[1])
        assert same(out.cpu(), want[2])


# ---------------------------------------------------------------------------
# reorder and copy
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B,K,width", [(1, 1, 3), (5, 4, 40), (3, 32, 7), (64, 8, 300), (2, 5, 1)])
def test_reorder(backend, B, K, width):
    rng = np.random.default_rng([B, K])
    table = rng.permutation(B * K * width).reshape(B * K, width).astype(np.int32)
    for parents in (rng.integers(0, K, (B, K)), np.zeros((B, K)), np.tile(np.arange(K)[::-1], (B, 1)),
                    rng.integers(-2, K + 2, (B, K))):
        parents = parents.astype(np.int32)
        out, src = torch.full((B * K, width), 99, dtype=torch.int32, device="cuda"), i32([99] * (B * K))
        backend.dev_beam_reorder(cuda(table), cuda(parents), out, src)
        want = reorder(table, parents)
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(src.cpu().numpy(), want[1])
        # no page is lost, none is had twice
        assert np.array_equal(np.sort(out.cpu().numpy(), None), np.sort(table, None))


POOLS = [(f, h, d, p) for f in ("f32", "bf16", "fp8", "int8", "fp4") for h, d, p in ((5, 128, 16), (2, 80, 32), (3, 34, 7),
                                                                                   (1, 2, 1), (2, 512, 16))]


@pytest.mark.parametrize("fmt,hkv,d,page", POOLS)
def test_copy(backend, fmt, hkv, d, page):
    """Codes and scales byte by byte; shared pages, missing pages, rows outside the
    window and every other page untouched."""
    say(f"copy {fmt} {hkv}/{d} page {page}")
    rng = np.random.default_rng([ord(c) for c in fmt] + [hkv, d, page])
    n, rows = 7, 90
    width = pages_of(rows, page)
    table = rng.permutation(n * width + 2)[: n * width].reshape(n, width).astype(np.int32)
    kv = PagedKV(n * width + 2, page, hkv, d, fmt)
    for t in (kv.k, kv.v, kv.k_scales, kv.v_scales):
        if t is not None:
            t.view(torch.uint8).random_(0, 256)
    lens = np.array([rows, rows, 33, 0, rows, 1 << 30, 50])
    starts = np.array([0, 0, 10, 0, 40, 0, -3])
    src = np.array([-1, 0, 0, 0, 6, 5, 7])  # 5 is itself, 6 has none
    src[5], src[6] = 5, n
    table[1, 0] = table[0, 0]
    if width > 2:
        table[2, 1], table[6, 2] = -1, n * width + 2
    before = {k: getattr(kv, k) for k in ("k", "v", "k_scales", "v_scales")}
    want = {k: t.view(torch.uint8).cpu().numpy().copy() for k, t in before.items() if t is not None}
    for s in range(n):
        if not 0 <= src[s] < n or src[s] == s:
            continue
        for t in range(max(starts[s], 0), min(lens[s], width * page)):
            a, b = table[src[s], t // page], table[s, t // page]
            if not (0 <= a < n * width + 2 and 0 <= b < n * width + 2):
                continue
            for k, w in want.items():
                r = w.reshape(n * width + 2, hkv, page, -1)
                r[b, :, t % page] = r[a, :, t % page]
    backend.dev_paged_copy(kv, i32(table), i32(src), i32(lens), starts=i32(starts))
    for k, w in want.items():
        assert np.array_equal(before[k].view(torch.uint8).cpu().numpy(), w), k
    # without starts, whole sequences: the others' bytes stay
    src = np.full(n, -1)
    src[3] = 1
    for t in range(rows):
        for w in want.values():
            r = w.reshape(n * width + 2, hkv, page, -1)
            r[table[3, t // page], :, t % page] = r[table[1, t // page], :, t % page]
    backend.dev_paged_copy(kv, i32(table), i32(src), i32([rows] * n))
    for k, w in want.items():
        assert np.array_equal(before[k].view(torch.uint8).cpu().numpy(), w), k


def test_copy_odd_address(backend):
    """A pool at an odd address, in bytes."""
    raw = torch.zeros(2, 4 * 2 * 16 * 32 + 1, dtype=torch.int8, device="cuda").random_(-128, 128)
    k, v = (raw[i, 1:].view(4, 2, 16, 32) for i in range(2))
    sc = torch.rand(2, 4, 2, 16, device="cuda")
    kv = PagedKV.from_tensors(k, v, sc[0], sc[1])
    want = k[3].clone()
    backend.dev_paged_copy(kv, i32([[3, 1], [0, 2]]), i32([-1, 0]), i32([16, 16]))
    assert torch.equal(k[0], want) and torch.equal(sc[1, 0], sc[1, 3])


def test_python_refusals(backend):
    kv = PagedKV(4, 16, 1, 32, "fp4")
    table, n = i32([[0, 1], [2, 3]]), i32([1, 2])
    logits, z = torch.zeros(2, 2, 50, device="cuda"), torch.zeros(2, 2, device="cuda")
    t = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    ws = backend.beam_workspace(2, 2, 50, 2)
    one = i32([1])
    for bad, error in [
        (lambda: backend.dev_paged_copy(kv, table.long(), n, n), TypeError),
        (lambda: backend.dev_paged_copy(kv, table[0], n, n), InvalidShape),
        (lambda: backend.dev_paged_copy(kv, table, n[:1], n), InvalidShape),
        (lambda: backend.dev_beam_select(logits.half(), z, t, t.clone(), z.clone(), ws), TypeError),
        (lambda: backend.dev_beam_select(logits.transpose(0, 1), z, t, t.clone(), z.clone(), ws), TypeError),
        (lambda: backend.dev_beam_select(logits.transpose(1, 2), z, t, t.clone(), z.clone(), ws), (TypeError, InvalidShape)),
        (lambda: backend.dev_beam_select(logits, z, t, t, z.clone(), ws), InvalidShape),
        (lambda: backend.dev_beam_select(logits, z, t, t.clone(), z, ws), InvalidShape),
        (lambda: backend.dev_beam_select(logits, z, t, t.clone(), z.clone(), ws[:64]), InvalidShape),
        (lambda: backend.dev_beam_select(logits, z, t, t.clone(), z.clone(), ws, done=z.byte()), InvalidConfig),
        (lambda: backend.dev_beam_reorder(table, t, table, n), (InvalidShape, TypeError)),
        (lambda: backend.dev_paged_extend(table, n, n, n, one, 16, n, n, i32([0, 0, 0]), n, one), InvalidShape),
        (lambda: backend.dev_paged_extend(table, n, n, n, one, 16, i32([1]), i32([1]), i32([0, 0]), n.clone(), one.clone()),
         InvalidShape),
    ]:
        with pytest.raises(error):
            bad()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("fmt,layout", [("fp4", "half"), ("fp4", "interleaved"), ("f32", "half")])
def test_search(backend, fmt, layout, captured):
    """Beam search over two requests: prompts go through extend, the rotation and
    the append once, beams share their pages; each step extends, rotates,
    appends, attends, selects, reorders and copies.  Every step's attention is
    checked against the beams' own histories, which numpy keeps.  Captured: two
    steps in one graph, on two sets of lengths, replayed."""
    say(f"search {fmt} {layout} captured {captured}")
    rng = np.random.default_rng(5)
    B, K, V, hq, hkv, d, page, steps = 2, 3, 211, 6, 2, 64, 16, 8
    n, prompt, width = B * K, [37, 20], 5
    rope = Rope(d if fmt == "f32" else 32, 500000.0, layout, scaling="parts", factor=4.0, original=16, beta=8.0)
    kv = PagedKV(n * width + 4, page, hkv, d, fmt)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    free = cuda(rng.permutation(kv.n_pages).astype(np.int32))
    count = [i32([kv.n_pages]), i32([0])]
    emb = [cuda((0.7 * rng.standard_normal((V, h * d))).astype(np.float32)) for h in (hq, hkv, hkv)]
    head = cuda((rng.standard_normal((hq * d, V)) / 8).astype(np.float32))
    # a request's beams start from one prompt
    history = [[list(p)] * K for p in (rng.integers(0, V, m) for m in prompt)]

    def rows_of(tokens, positions):
        """q, k, v of tokens as the cache and the attention have them (from the device's own rotation)."""
        t = torch.as_tensor(np.array(tokens)).cuda()
        q, k, v = (e[t].view(len(tokens), -1, d).clone() for e in emb)
        backend.dev_rope(rope, q, k, i32(positions))
        keep = (lambda x: values(*encode(x))) if fmt == "fp4" else (lambda x: x)
        return q.cpu().numpy(), keep(k.cpu().numpy()), keep(v.cpu().numpy())

    # prompts: the first beam of each request, then the others share its full pages and copy the rest
    lens = [i32([0] * n), i32([0] * n)]
    first = np.zeros(n, np.int32)
    first[::K] = prompt
    total = int(first.sum())
    seqs, pos = (torch.zeros(total, dtype=torch.int32, device="cuda") for _ in range(2))
    off = i32([0] * (n + 1))
    backend.dev_paged_extend(table, lens[0], i32(first), free, count[0], page, seqs, pos, off, lens[1], count[1])
    x = torch.as_tensor(np.concatenate([history[b][0] for b in range(B)])).cuda()
    q, k, v = (e[x].view(total, -1, d).clone() for e in emb)
    backend.dev_rope(rope, q, k, pos)
    backend.dev_paged_append(kv, None, k, v, None, pos, table, seqs=seqs)
    shared = [p // page for p in prompt]
    others = np.zeros(n, np.int32)
    have = np.zeros(n, np.int32)
    for b in range(B):
        for j in range(1, K):
            table[b * K + j, :shared[b]] = table[b * K, :shared[b]]
            have[b * K + j] = shared[b] * page
            others[b * K + j] = prompt[b] - shared[b] * page
        have[b * K] = prompt[b]
    backend.dev_paged_extend(table, i32(have), i32(others), free, count[1], page, torch.zeros_like(seqs),
                             torch.zeros_like(pos), off, lens[0], count[0])
    src = i32([-1 if s % K == 0 else s // K * K for s in range(n)])
    starts = i32([shared[s // K] * page for s in range(n)])
    backend.dev_paged_copy(kv, table, src, lens[0], starts=starts)
    assert lens[0].tolist() == [p for p in prompt for _ in range(K)]

    tables = [table, torch.empty_like(table)]
    tokens = [cuda(np.array([[h[-1] for h in r] for r in history], np.int32)), torch.zeros(B, K, dtype=torch.int32, device="cuda")]
    scores = [torch.full((B, K), -float("inf"), device="cuda"), torch.zeros(B, K, device="cuda")]
    scores[0][:, 0] = 0
    done = [torch.zeros(B, K, dtype=torch.uint8, device="cuda") for _ in range(2)]
    parents = [torch.zeros(B, K, dtype=torch.int32, device="cuda") for _ in range(2)]
    outs = [torch.zeros(n, hq, d, device="cuda") for _ in range(2)]
    one, eos = i32([1] * n), 7
    ws, ws2 = backend.paged_workspace(kv, n, hq), backend.beam_workspace(B, K, V, K)
    seqs, pos, off = i32([0] * n), i32([0] * n), i32([0] * (n + 1))
    q, k, v = (torch.zeros(n, h, d, device="cuda") for h in (hq, hkv, hkv))

    def step(a, b):
        backend.dev_paged_extend(tables[a], lens[a], one, free, count[a], page, seqs, pos, off, lens[b], count[b])
        t = tokens[a].view(-1)
        for to, e in zip((q, k, v), emb):
            torch.index_select(e, 0, t, out=to.view(n, -1))
        backend.dev_rope(rope, q, k, pos)
        backend.dev_paged_append(kv, None, k, v, None, pos, tables[a])
        backend.dev_paged_decode_attention(kv, q, tables[a], lens[b], outs[a], ws)
        logits = (outs[a].view(n, -1)[:, :, None] * head).sum(1).view(B, K, V)
        backend.dev_beam_select(logits, scores[a], tokens[b], parents[b], scores[b], ws2, done=done[a], eos=eos,
                                done_out=done[b])
        backend.dev_beam_reorder(tables[a], parents[b], tables[b], src)
        backend.dev_paged_copy(kv, tables[b], src, lens[b], starts=starts)

    def check(a, b, before):
        """outs[a] is the attention of the histories with the token that tokens[a] held."""
        got, length = outs[a].cpu().numpy(), lens[b].cpu().numpy()
        par, tok = parents[b].cpu().numpy(), tokens[b].cpu().numpy()
        grown = []
        for r in range(B):
            for j in range(K):
                # the last prompt token is appended a second time by the first step
                h = history[r][j] + [int(before[r, j])]
                assert length[r * K + j] == len(h)
                qr, kr, vr = rows_of(h, range(len(h)))
                want, mag, size = attention(qr[-1], kr, vr)
                bound = attention_bound(len(h), d, mag, size)
                assert float((np.abs(got[r * K + j] - want) / bound).max()) <= 1, (r, j)
                grown.append(h)
        for r in range(B):
            history[r] = [grown[r * K + par[r, j]] for j in range(K)]
        assert (par >= 0).all() and (par < K).all() and (tok >= 0).all() and (tok < V).all()

    # the two halves of a graph leave what each half's check needs: one half at a time is checked
    if not captured:
        for i in range(steps):
            a, b = i % 2, 1 - i % 2
            before = tokens[a].cpu().numpy()
            step(a, b)
            check(a, b, before)
    else:
        graphs = []
        state = [*tables, *lens, *count, *tokens, *scores, *done, *parents, kv.k, kv.v, free]
        state += [t for t in (kv.k_scales, kv.v_scales) if t is not None]
        saved = [t.clone() for t in state]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(0, 1)
            step(1, 0)
        torch.cuda.current_stream().wait_stream(s)
        for t, old in zip(state, saved):
            t.copy_(old)
        for a in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step(a, 1 - a)
            graphs.append(g)
        for t, old in zip(state, saved):
            t.copy_(old)
        for i in range(steps):
            a, b = i % 2, 1 - i % 2
            before = tokens[a].cpu().numpy()
            graphs[a].replay()
            torch.cuda.synchronize()
            check(a, b, before)
    assert all(len(h) == prompt[r] + steps for r in range(B) for h in history[r])
    # the rows that the beams' tables name are the histories' rows
    end = steps % 2
    most = max(prompt) + steps
    back = [torch.zeros(n, hkv, most, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, tables[end], lens[end], *back)
    for r in range(B):
        for j in range(K):
            _, kr, vr = rows_of(history[r][j], range(len(history[r][j])))
            for o, w in zip(back, (kr, vr)):
                assert same(o[r * K + j, :, :len(w)].cpu().numpy().transpose(1, 0, 2), w)


# ---------------------------------------------------------------------------
# long rows of many requests, streams, threads
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("V", [20001, 33000])
def test_select_many_rows(backend, V):
    """So many rows that a workgroup takes a whole one, in several turns: ties over
    the turns' borders, floods of equal logits early and late, masks that leave
    the first turn, all turns but the last, or a few tokens."""
    B, K, k = 40, 26, 20
    rng = np.random.default_rng(V)
    logits = (2 * rng.standard_normal((B, K, V))).astype(np.float32)
    logits[0] = 1.5
    logits[1, :, :4096] = -np.inf
    logits[2, :, : V - 30] = -np.inf
    logits[3] = -np.inf
    logits[3, :, [5, 4095, 4096, 4097, 8191, 8192, V - 1]] = 2.0
    logits[4, :, 4000:4200] = 40.0
    logits[5, :, -300:] = 40.0
    logits[6, :, ::7] = 9.25
    logits[7] = np.sort(logits[7], -1)
    logits[8] = np.sort(logits[8], -1)[:, ::-1]
    logits[9] = rng.integers(-3, 4, (K, V))
    logits[10, :, 200:] = -np.inf
    logits[10, :, :200] = 0.5
    logits[11, 3, 9000], logits[11, 4, V - 1] = np.nan, np.inf
    scores = (-3 * rng.random((B, K))).astype(np.float32)
    scores[12] = -1.25
    logits[12] = logits[12, 0]
    check_select(backend, logits, scores, k)
    done = (rng.random((B, K)) < 0.3).astype(np.uint8)
    check_select(backend, logits, scores, k, done, 4096)


def test_streams_of_their_own(backend):
    """The calls on two streams at once, each with its own buffers, by the stream
    that is current and by the argument: the results of one after the other."""
    rng = np.random.default_rng(77)
    V, K = 9001, 4
    sides = []
    for i in range(2):
        s = {"logits": cuda((2 * rng.standard_normal((8, K, V))).astype(np.float32)), "scores": torch.zeros(8, K, device="cuda"),
             "tokens": i32(np.zeros((8, K))), "parents": i32(np.zeros((8, K))), "out": torch.zeros(8, K, device="cuda"),
             "ws": backend.beam_workspace(8, K, V, K), "kv": PagedKV(200, 16, 2, 64, "fp4"),
             "table": cuda(rng.permutation(200)[:192].reshape(32, 6).astype(np.int32)), "lens": i32([90] * 32),
             "to": torch.zeros(32, 6, dtype=torch.int32, device="cuda"), "src": i32([0] * 32),
             "q": torch.randn(32, 6, 64, device="cuda"), "pos": i32(rng.integers(0, 1 << 20, 32)), "rot": torch.zeros(32, 6, 64, device="cuda")}
        for t in (s["kv"].k, s["kv"].v):
            t.random_(0, 256)
        for t in (s["kv"].k_scales, s["kv"].v_scales):
            t.random_(120, 130)
        sides.append(s)
    rope = Rope(64, 10000.0, "interleaved")

    def run(s, stream=None):
        backend.dev_beam_select(s["logits"], s["scores"], s["tokens"], s["parents"], s["out"], s["ws"], stream=stream)
        backend.dev_beam_reorder(s["table"], s["parents"], s["to"], s["src"], stream=stream)
        backend.dev_paged_copy(s["kv"], s["to"], s["src"], s["lens"], stream=stream)
        backend.dev_rope(rope, s["q"], None, s["pos"], s["rot"], stream=stream)

    keys = ("tokens", "parents", "out", "to", "src", "rot")
    pools = [(s["kv"].k.clone(), s["kv"].v.clone()) for s in sides]
    want = []
    for s in sides:
        run(s)
        torch.cuda.synchronize()
        want.append([s[k].clone() for k in keys] + [s["kv"].k.clone(), s["kv"].v.clone()])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, (k, v) in zip(sides, pools):
            s["kv"].k.copy_(k)
            s["kv"].v.copy_(v)
            for n in keys:
                s[n].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            run(sides[0])
        run(sides[1], streams[1])
        torch.cuda.synchronize()
        for s, w in zip(sides, want):
            for got, exp in zip([s[k] for k in keys] + [s["kv"].k, s["kv"].v], w):
                assert torch.equal(got, exp)


def test_two_threads(backend):
    """Two host threads make the calls side by side, on streams of their own."""
    import threading

    V, K, n = 3001, 3, 50
    rope = Rope(32, 10000.0)
    wrong = []

    def work(seed):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                g = torch.Generator(device="cuda").manual_seed(seed)
                x = torch.randn(2, K, V, device="cuda", generator=g)
                q = torch.randn(n, 2, 48, device="cuda", generator=g)
                p = torch.randint(0, 9999, (n,), device="cuda", dtype=torch.int32, generator=g)
                ws, first = backend.beam_workspace(2, K, V, K), None
                for _ in range(30):
                    t, par = (torch.zeros(2, K, dtype=torch.int32, device="cuda") for _ in range(2))
                    out, rot = torch.zeros(2, K, device="cuda"), torch.zeros_like(q)
                    backend.dev_beam_select(x, torch.zeros(2, K, device="cuda"), t, par, out, ws)
                    backend.dev_rope(rope, q, None, p, rot)
                    got = [y.clone() for y in (t, par, out, rot)]
                    stream.synchronize()
                    if first is not None and not all(torch.equal(a, b) for a, b in zip(first, got)):
                        wrong.append(seed)
                    first = got
        except Exception as e:  # noqa: BLE001 (reported by the test)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


@pytest.mark.parametrize("n", [1, 64])
def test_extend_and_release_captured(backend, n):
    """One graph of an extend and a release, replayed on other counts."""
    rng = np.random.default_rng(n)
    page, width, free = 16, 8, 8 * n
    t = Tables(rng, rng.integers(0, 60, n), width, page, free, cap=free + 8 * n)
    table, lens, stack, count = cuda(t.table), cuda(t.lens), cuda(t.free), i32([free])
    new, which = i32([1] * n), torch.zeros(n, dtype=torch.uint8, device="cuda")
    seqs, pos, off = i32([0] * 40 * n), i32([0] * 40 * n), i32([0] * (n + 1))
    l2, c2, l3, c3 = i32([0] * n), i32([0]), i32([0] * n), i32([0])

    def both():
        backend.dev_paged_extend(table, lens, new, stack, count, page, seqs, pos, off, l2, c2)
        backend.dev_paged_release(table, l2, which, stack, c2, page, l3, c3)

    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(g):
        both()
    for i in range(4):
        table.copy_(cuda(t.table))
        stack.copy_(cuda(t.free))
        more, gone = rng.integers(0, 40, n), (rng.random(n) < 0.5).astype(np.uint8)
        new.copy_(i32(more))
        which.copy_(cuda(gone))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        a = extend(t.table, t.lens, more, t.free, free, page, 40 * n)
        b = release(a[0], a[1], gone, None, t.free, a[2], page)
        for got, w in zip((seqs, pos, off, l2, table, l3, stack, c3), (a[3], a[4], a[6], a[1], b[0], b[1], b[2], [b[3]])):
            assert np.array_equal(got.cpu().numpy(), w)


def test_workspace_of_the_largest_batch(backend):
    """A workspace made once for 16 requests of 8 beams, as requests end: fewer rows
    are cut into more parts."""
    K, V = 8, 40000
    ws = backend.beam_workspace(16, K, V, K)
    rng = np.random.default_rng(15)
    logits = (3 * rng.standard_normal((16, K, V))).astype(np.float32)
    scores = (-4 * rng.random((16, K))).astype(np.float32)
    for B, beams, k in ((16, K, K), (15, K, K), (14, K, K), (9, K, 5), (3, K, K), (1, K, K), (1, 1, 8), (16, 3, 3)):
        say(f"select {B}x{beams} k {k} in the workspace of 16x8")
        x, s = logits[:B, :beams], scores[:B, :beams]
        tokens, parents, _, _, gap = select(x, s, k)
        assert gap > 2.0 ** -16
        got = run_select(backend, cuda(x), cuda(s), k, ws=ws)
        assert np.array_equal(got[0], tokens) and np.array_equal(got[1], parents)


# Any vocabulary: a part's sum is joined in 64 bits every 16 terms of a thread, whose
# additions are five roundings (5 * 2^-24).  A term is a product of factors exp(d):
# its own, from a reference that is at most 2 below the largest logit so far, and
# one each time the reference rises by more than 2, or two threads, waves or parts
# are joined.  The |d| of one term come to its distance from the largest logit and
# at most 2 + 4, on the mean over the softmax ln V + 6 < 27 (V <= 2^30); each is off
# by 3 |d| 2^-24 + 2^-23, and there are at most 27 / 2 + 3 of them: 81 + 33 + 5 = 119
# times 2^-24, under 2^-17.
LSE = 2.0 ** -17


def flood(V, part):
    """Of each `part` logits the first 1024 are 0, and all others so small that an
    fp32 sum of 1 does not notice one of them: exp is just under 2^-24."""
    x = torch.full((V // part, part), -24 * float(np.log(2)) - 1e-5, device="cuda")
    x[:, :1024] = 0
    return x.view(V)


def lse64(x):
    return float(torch.logsumexp(x.double(), -1))


def test_select_sums_of_a_large_vocabulary(backend):
    """2^25 logits in 64 parts: what half a million small ones add decides between
    two beams."""
    V = 1 << 25
    logits = torch.full((1, 2, V), -float("inf"), device="cuda")
    logits[0, 0] = flood(V, V // 64)
    logits[0, 1, :1 << 16] = 0
    want = -np.array([lse64(logits[0, 0]), np.log(65536.0)])
    assert want[1] - want[0] > 2 * LSE
    tokens, parents, got, _ = run_select(backend, logits, torch.zeros(1, 2, device="cuda"), 2)
    assert parents.tolist() == [[1, 1]] and tokens.tolist() == [[0, 1]]
    tokens, parents, got, _ = run_select(backend, logits, torch.tensor([[1.0, 0.0]], device="cuda"), 2)
    assert parents.tolist() == [[0, 0]] and tokens.tolist() == [[0, 1]]
    assert np.abs(got - (1 + want[0])).max() <= LSE + 12 * 2.0 ** -24


@pytest.mark.parametrize("V", [1 << 18, (1 << 18) - 1])
def test_select_sums_of_whole_rows(backend, V):
    """1024 rows and more: a row is one part, with 256 terms a thread's sum."""
    x = flood(1 << 18, 1 << 18)[:V]
    logits = x.expand(128, 8, V).contiguous()
    scores = -torch.arange(8, device="cuda", dtype=torch.float32).expand(128, 8).contiguous()
    tokens, parents, got, _ = run_select(backend, logits, scores, 4)
    assert (parents == 0).all() and (tokens == np.arange(4)).all()
    assert np.abs(got + lse64(x)).max() <= LSE + 8 * 2.0 ** -24


@pytest.mark.parametrize("step", [2.0 ** -20, 2.0 ** -16, 2.0 ** -13])
@pytest.mark.parametrize("B,V", [(1, 1 << 22), (1024, 1 << 16)])
def test_select_sums_of_rising_logits(backend, B, V, step):
    """Each logit is larger than those before it, and the other way round."""
    up = torch.arange(V, device="cuda", dtype=torch.float32) * step
    for x in (up, up.flip(0)):
        logits = x.expand(B, 1, V).contiguous()
        tokens, _, got, _ = run_select(backend, logits, torch.zeros(B, 1, device="cuda"), 3)
        best = torch.topk(x, 3)
        assert (tokens == best.indices.cpu().numpy()).all()
        want = best.values.double().cpu().numpy() - lse64(x)
        assert (np.abs(got - want) <= LSE + np.abs(want) * 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", ["fp4", "fp8", "int8"])
def test_copies_on_two_streams(backend, fmt):
    """Copies of two pools on two streams at once: codes and scales byte by byte."""
    rng = np.random.default_rng(5)
    n, page, width, rows = 32, 16, 6, 90
    sides = []
    for i in range(2):
        kv = PagedKV(n * width + 8, page, 2, 64, fmt)
        table = rng.permutation(n * width + 8)[:n * width].reshape(n, width).astype(np.int32)
        src = np.full(n, -1, np.int32)
        src[1::2] = rng.integers(0, n // 2, n // 2) * 2  # odd sequences from even ones
        tensors = [kv.k, kv.v, kv.k_scales, kv.v_scales]
        for t in tensors:
            t.view(torch.uint8).random_(0, 256)
        first = [t.view(torch.uint8).cpu().numpy().copy() for t in tensors]
        want = [x.copy() for x in first]
        for s in range(1, n, 2):
            for t in range(3, rows):
                a, b = table[src[s], t // page], table[s, t // page]
                for x, w in zip(first, want):
                    # [pages, kv heads, page, bytes of a row] (a scale's four bytes as a row of their own)
                    x, w = (y.reshape(n * width + 8, 2, page, -1) for y in (x, w))
                    w[b, :, t % page] = x[a, :, t % page]
        sides.append((kv, cuda(table), i32(src), tensors, first, want))
    lens, starts = i32([rows] * n), i32([3] * n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for _, _, _, tensors, first, _ in sides:
            for t, x in zip(tensors, first):
                t.view(torch.uint8).copy_(cuda(x))
        torch.cuda.synchronize()
        for (kv, table, src, *_), stream in zip(sides, streams):
            backend.dev_paged_copy(kv, table, src, lens, starts, stream=stream)
        torch.cuda.synchronize()
        for _, _, _, tensors, _, want in sides:
            for t, w in zip(tensors, want):
                assert np.array_equal(t.view(torch.uint8).cpu().numpy(), w)


@pytest.mark.parametrize("fmt", ["fp4", "bf16"])
def test_steps_from_a_fused_projection(backend, fmt):
    """A server's step on slices of one projection's output, as the integration
    guide has it: the results of the same calls on tensors of their own."""
    batch, hq, hkv, d, page, width = 3, 8, 2, 64, 16, 4
    rope = Rope(d, 10000.0, scaling="parts", factor=8.0, original=4096, magnitude=1.2)
    sides = []
    for _ in range(2):
        kv = PagedKV(batch * width, page, hkv, d, fmt)
        sides.append([kv, i32(np.full((batch, width), -1)), i32(np.arange(batch * width)), i32([0, 20, 16]), i32([batch * width])])
        table, free, lens, count = sides[-1][1:]
        # pages of the rows that are there
        for s, n in enumerate(lens.tolist()):
            for p in range(pages_of(n, page)):
                count -= 1
                table[s, p] = free[count.item()]
    new, seqs, positions, offsets = i32([1] * batch), i32([0] * batch), i32([0] * batch), i32([0] * (batch + 1))
    ws = backend.paged_workspace(sides[0][0], batch, hq)
    for _ in range(5):
        qkv = torch.randn(batch, hq + 2 * hkv, d, device="cuda")
        outs = []
        for fused, side in ((True, sides[0]), (False, sides[1])):
            kv, table, free, lens, count = side
            lens2, count2 = torch.empty_like(lens), torch.empty_like(count)
            backend.dev_paged_extend(table, lens, new, free, count, page, seqs, positions, offsets, lens2, count2)
            q, k, v = qkv[:, :hq], qkv[:, hq:-hkv], qkv[:, -hkv:].contiguous()
            if fused:
                to = torch.empty(batch, hq, d, device="cuda"), torch.empty(batch, hkv, d, device="cuda")
                backend.dev_rope(rope, q, k, positions, *to)
                q, k = to
            else:
                q, k = q.contiguous(), k.contiguous()
                backend.dev_rope(rope, q, k, positions)
            backend.dev_paged_append(kv, None, k, v, None, positions, table, seqs=seqs)
            out = torch.empty_like(q)
            backend.dev_paged_decode_attention(kv, q, table, lens2, out, ws)
            side[3:] = lens2, count2
            outs.append(out)
        assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    assert torch.equal(sides[0][0].k.view(torch.uint8), sides[1][0].k.view(torch.uint8)) and sides[0][3].tolist() == [5, 25, 21]
