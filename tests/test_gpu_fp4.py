"""The paged cache's 4-bit rows on the GPU: append and read bit by bit, decode
attention against 64 bits, and a run of them as a server would use them."""
import numpy as np
import pytest
import torch

from fp4_common import (Pool4, attention, attention_bound, encode, groups, i32, rotate, same, values)

pytestmark = pytest.mark.gpu

THETA = 500000.0
SHAPES = [(20, 5, 128, 16), (8, 8, 64, 16), (14, 2, 80, 32), (4, 4, 96, 64), (16, 2, 256, 128), (6, 3, 144, 16),
          (3, 1, 2, 1), (2, 1, 6, 5), (6, 3, 34, 7), (4, 2, 136, 48), (5, 5, 510, 16), (2, 2, 512, 8)]


def say(msg):
    print(f"[gpu case] {msg}", flush=True)


def rng_of(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check_rows(pool, kv, where, rows):
    """The pool's bytes: these rows' codes and exponents at `where` (page, row), all else as it was."""
    for n in "kv":
        codes, exps = encode(rows[n])
        want, want_e = pool.codes[n].copy(), pool.exps[n].copy()
        want[where[0], :, where[1]], want_e[where[0], :, where[1]] = codes, exps
        assert np.array_equal(getattr(kv, n).cpu().numpy(), want), n
        assert np.array_equal(getattr(kv, n + "_scales").cpu().numpy(), want_e), n


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("hq,hkv,d,page", SHAPES)
def test_append(backend, hq, hkv, d, page, aligned):
    """Ragged tokens of three sequences in no order, with rotation: codes and
    exponents bit by bit, and no other row touched; unaligned inputs too."""
    say(f"append fp4 {hq}/{hkv}/{d} page {page} aligned {aligned}")
    rng = rng_of(hq, hkv, d, page)
    width = -(-40 // page)
    pool = Pool4(rng, [width * page] * 3, hkv, d, page)
    where = [(s, t) for s, t0, n in ((0, 0, 5), (1, 11, 21), (2, 39, 1)) for t in range(t0, t0 + n)]
    rng.shuffle(where)
    seqs, pos = (np.array(x) for x in zip(*where))
    n = len(where)
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (hq, hkv, hkv))
    cos, sin = backend.rope_table(width * page, d, THETA)
    cosn, sinn = cos.cpu().numpy(), sin.cpu().numpy()
    kv = pool.device()

    def place(x):
        if aligned:
            return cuda(x)
        y = torch.empty(x.size + 1, device="cuda")[1:].view(x.shape)
        return y.copy_(cuda(x))

    q_out = torch.full((n, hq, d), 7.0, device="cuda")
    backend.dev_paged_append(kv, place(q), place(k), place(v), q_out, i32(pos), i32(pool.table), cos, sin,
                             seqs=i32(seqs))
    torch.cuda.synchronize()
    assert same(q_out.cpu(), rotate(q, cosn[pos], sinn[pos]))
    check_rows(pool, kv, (pool.table[seqs, pos // page], pos % page), {"k": rotate(k, cosn[pos], sinn[pos]), "v": v})


@pytest.mark.parametrize("d", [128, 64, 80, 22, 512])
def test_append_extreme_rows(backend, d):
    """Zeros, powers of two and the values between two codes, tiny and huge rows,
    groups that hold an infinity or a NaN."""
    rng = rng_of("extreme", d)
    n, page = 24, 16
    x = rng.standard_normal((n, 1, d)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= np.float32(1e-42)
    x[3] *= np.float32(1e-30)
    x[4] = np.float32(3.4028235e38)
    x[5] *= np.float32(1e38) / np.abs(x[5]).max()
    x[6, 0, 0] = np.inf
    x[7, 0, d - 1] = -np.inf
    x[8, 0, d // 2] = np.nan
    x[9] = np.nan
    x[10] = np.resize(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6], np.float32), d)
    x[11] = -x[10] * np.float32(2.0 ** -40)
    x[12] = np.resize(np.array([1.75, 1.7499999, 1.5, 1.0], np.float32), d)
    x[13] = np.float32(1.7499999) * np.float32(2.0 ** 60)
    x[14] = 0
    x[14, 0, d - 1] = np.float32(1e-45)
    x[15:] *= np.exp(4 * rng.standard_normal((n - 15, 1, d))).astype(np.float32)
    pool = Pool4(rng, [n], 1, d, page)
    kv = pool.device()
    backend.dev_paged_append(kv, None, cuda(x), cuda(x[::-1]), None, i32(range(n)), i32(pool.table), seqs=i32([0] * n))
    at = np.arange(n)
    check_rows(pool, kv, (pool.table[0, at // page], at % page), {"k": x, "v": x[::-1]})
    out = [torch.zeros(1, 1, n, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, i32(pool.table), i32([n]), *out)
    for o, w in zip(out, (x, x[::-1])):
        assert same(o[0].cpu().numpy().transpose(1, 0, 2), values(*encode(w)))


@pytest.mark.parametrize("hq,hkv,d,page", SHAPES)
def test_read(backend, hq, hkv, d, page):
    """Windows of ragged sequences: the codes' values; other rows stay, pages that
    are not there read as zeros; every exponent, NaN's among them."""
    say(f"read fp4 {hkv}/{d} page {page}")
    rng = rng_of("read", hkv, d, page)
    lens, starts, cap = [70, 0, 33, 1], [3, 0, 33, 0], 75
    pool = Pool4(rng, lens, hkv, d, page)
    for n in "kv":
        pool.exps[n] = rng.integers(0, 256, pool.exps[n].shape).astype(np.uint8)
    if pool.table.shape[1] > 2:
        pool.table[0, 1] = -1
    kv = pool.device()
    outs = [torch.full((4, hkv, cap, d), 3.0, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, i32(pool.table), i32(lens), *outs, starts=i32(starts))
    for n, o in zip("kv", outs):
        o = o.cpu().numpy()
        for s, (a, b) in enumerate(zip(starts, lens)):
            rows, there = pool.rows(n, s)
            want = np.where(there[:, None, None], rows, 0)[a:]
            assert same(o[s, :, :b - a].transpose(1, 0, 2), want)
            assert (o[s, :, b - a:] == 3).all()


def room(n_seqs, hkv, page, wide):
    """Pages of a table with room for more than 1024 units of 128 rows, from which on up to four heads share columns."""
    return 150000 // (n_seqs * hkv * page) + 1 if wide else 0


def run_decode(be, pool, hq, lens, seed=1, q=None, out=None):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((len(lens), hq, pool.d)).astype(np.float32) if q is None else q
    kv = pool.device()
    ws = be.paged_workspace(kv, len(lens), hq)
    out = torch.full((len(lens), hq, pool.d), 9.0, device="cuda") if out is None else out
    be.dev_paged_decode_attention(kv, cuda(q), i32(pool.table), i32(lens), out, ws)
    torch.cuda.synchronize()
    return q, out.cpu().numpy()


def check_decode(pool, q, got, lens):
    for s, n in enumerate(lens):
        k, there = pool.rows("k", s, n)
        v, _ = pool.rows("v", s, n)
        want, mag, size = attention(q[s], k[there], v[there])
        bound = attention_bound(max(int(there.sum()), 1), pool.d, mag, size)
        off = np.abs(got[s] - want)
        assert (off <= bound).all(), (s, n, float((off / bound).max()))


DECODE = SHAPES + [(16, 1, 128, 16), (16, 1, 256, 16), (17, 1, 64, 16), (40, 2, 48, 32), (4, 4, 16, 16), (12, 4, 240, 48),
                   (20, 5, 112, 64)]


@pytest.mark.parametrize("hq,hkv,d,page", DECODE)
def test_decode(backend, hq, hkv, d, page):
    say(f"decode fp4 {hq}/{hkv}/{d} page {page}")
    lens = [1, 300, 0, 33, 129, 16]
    pool = Pool4(rng_of("decode", hq, hkv, d, page), lens, hkv, d, page)
    q, got = run_decode(backend, pool, hq, lens)
    check_decode(pool, q, got, lens)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [7], [4096], [5001], [20000, 3],
                                  [0] * 70 + [300] + [0] * 60 + [5], [129] * 65, [64, 1, 2000, 0, 777]])
def test_decode_batches(backend, lens):
    say(f"decode fp4 batch of {len(lens)}, longest {max(lens)}")
    pool = Pool4(rng_of("batch", lens), lens, 5, 128, 16)
    q, got = run_decode(backend, pool, 20, lens)
    check_decode(pool, q, got, lens)


@pytest.mark.parametrize("hq,hkv,d,page,n", [(20, 5, 128, 16, 3000), (8, 8, 64, 64, 1500), (3, 1, 256, 16, 9000),
                                              (6, 3, 80, 32, 2500), (2, 1, 144, 16, 20000), (16, 2, 128, 16, 5000)])
def test_decode_large_tables(backend, hq, hkv, d, page, n):
    """Tables with room for many units, where up to four heads share columns:
    ragged lengths, long, short and none, in the same table."""
    say(f"decode fp4 {hq}/{hkv}/{d} up to {n} rows")
    lens = [n, 0, 1, n - 1, 700, n // 2 + 5, 33, n] + [129] * 4
    pool = Pool4(rng_of("large", hq, d, n), lens, hkv, d, page, width=max(-(-n // page), room(len(lens), hkv, page, True)))
    q, got = run_decode(backend, pool, hq, lens)
    check_decode(pool, q, got, lens)
    assert (got[1] == 0).all()
    few = [5, 0, 1, 0, 700, 3, 33, 2] + [129] * 4
    check_decode(pool, *run_decode(backend, pool, hq, few, q=q), few)


@pytest.mark.parametrize("hq,hkv,d,page,lens", [(12, 1, 80, 16, [30000]), (16, 1, 128, 64, [17, 21000]),
                                                (16, 1, 256, 16, [9000]), (4, 1, 64, 128, [40001]),
                                                (3, 1, 34, 7, [9000])])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_counts_every_row_once(backend, hq, hkv, d, page, lens, wide):
    """No score differs, so an output is its column's sum over the number of rows.
    The sum is of small whole numbers and halves, exact in fp32; what is left is
    the waves' and pieces' factors (powers of two, exact here) and one division:
    a reciprocal's rounding and a product's, 2^-23 together."""
    rng = rng_of("count", hq, d, lens)
    pool = Pool4(rng, lens, hkv, d, page, width=max(-(-max(lens) // page), room(len(lens), hkv, page, wide)))
    pool.exps["v"][:] = rng.integers(127, 129, pool.exps["v"].shape)
    q, got = run_decode(backend, pool, hq, lens, q=np.zeros((len(lens), hq, d), np.float32))
    for s, n in enumerate(lens):
        v, _ = pool.rows("v", s, n)
        total = v.astype(np.float64).sum(0)
        assert np.abs(v).sum(0).max() < 2 ** 23
        want = np.repeat(total / n, hq // hkv, 0)
        assert (np.abs(got[s] - want) <= np.abs(want) * 2.0 ** -22).all()


@pytest.mark.parametrize("d,page", [(128, 16), (128, 64), (80, 32), (10, 3)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_missing_pages_and_lengths(backend, d, page, wide):
    """Pages that are not there are left out; lengths outside the table are cut;
    NaN codes behind a sequence's last row, and in pages of others, do not show."""
    lens = [10 * page, 4 * page + 1, 3 * page, 2]
    pool = Pool4(rng_of("missing", d, page), lens, 2, d, page, width=max(10, room(4, 2, page, wide)))
    n_pages = pool.codes["k"].shape[0]
    for n in "kv":
        used = np.zeros(pool.exps[n].shape[:3], bool)
        for s, length in enumerate(lens):
            t = np.arange(length)
            used[pool.table[s, t // page], :, t % page] = True
        pool.exps[n][~used] = 255
    pool.table[0, 3], pool.table[0, 0], pool.table[1, 4] = -1, n_pages, -7
    pool.table[2, :] = -1
    asked = [10 * page, 4 * page + 1, 3 * page, 2]
    q, got = run_decode(backend, pool, 4, asked)
    check_decode(pool, q, got, asked)
    assert (got[2] == 0).all()
    q, got = run_decode(backend, pool, 4, [1 << 30, -5, 0, 2])
    check_decode(pool, q, got, [pool.table.shape[1] * page, 0, 0, 2])


@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (256, 16), (80, 32), (26, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_non_finite_groups_show(backend, d, page, wide):
    """A NaN group in V makes its columns NaN, one in K the heads that read it; no
    other sequence, head or column."""
    lens = [200, 200, 200]
    pool = Pool4(rng_of("nan", d), lens, 2, d, page, width=max(-(-200 // page), room(3, 2, page, wide)))
    g = groups(d) - 1
    pool.exps["v"][pool.table[0, 77 // page], 1, 77 % page, g] = 255
    pool.exps["k"][pool.table[1, 150 // page], 0, 150 % page, 0] = 255
    q, got = run_decode(backend, pool, 6, lens)
    nan = np.isnan(got)
    want = np.zeros_like(nan)
    want[0, 3:, 32 * g:] = True
    want[1, :3] = True
    assert np.array_equal(nan, want)
    check_decode(pool, q[2:], got[2:], [])
    k, _ = pool.rows("k", 2)
    v, _ = pool.rows("v", 2)
    w, mag, size = attention(q[2], k, v)
    assert (np.abs(got[2] - w) <= attention_bound(200, d, mag, size)).all()


@pytest.mark.parametrize("d,page", [(128, 16), (26, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_scores_of_any_size(backend, d, page, wide):
    """Scores hundreds apart, and groups of very different powers."""
    lens = [700, 90]
    pool = Pool4(rng_of("wide", d), lens, 2, d, page, width=max(-(-700 // page), room(2, 2, page, wide)), spread=6.0)
    q, got = run_decode(backend, pool, 4, lens)
    check_decode(pool, q, got, lens)


def test_decode_same_bits_workspace_and_graph(backend):
    """Captured once, replayed with other lengths and rows between; the same bits
    as an eager call; a workspace is ready again after each call."""
    hq, hkv, d, page = 20, 5, 128, 16
    pool = Pool4(rng_of("graph"), [3000, 800, 1], hkv, d, page)
    kv = pool.device()
    ws, ws2 = (backend.paged_workspace(kv, 3, hq) for _ in range(2))
    q = torch.randn(3, hq, d, device="cuda")
    table, lens = i32(pool.table), i32([10, 800, 0])
    out, eager = torch.empty_like(q), torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        backend.dev_paged_decode_attention(kv, q, table, lens, out, ws)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        backend.dev_paged_decode_attention(kv, q, table, lens, out, ws)
    for n in ([3000, 800, 1], [1, 1, 0], [2999, 0, 1], [3000, 800, 1]):
        lens.copy_(i32(n))
        q.normal_()
        g.replay()
        backend.dev_paged_decode_attention(kv, q, table, lens, eager, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check_decode(pool, q.cpu().numpy(), out.cpu().numpy(), n)


@pytest.mark.parametrize("hq,hkv,d,page", [(20, 5, 128, 16), (6, 2, 80, 32), (4, 2, 34, 5)])
def test_serving_run(backend, hq, hkv, d, page):
    """Prompts of three sequences appended, then tokens one by one with their
    attention, against the numpy cache; and the rows read back for a prefill."""
    say(f"serving fp4 {hq}/{hkv}/{d} page {page}")
    from bitnetrs_amd import PagedKV

    rng = rng_of("serve", d)
    lens, width = [50, 1, 23], -(-70 // page)
    order = rng.permutation(3 * width)
    table = order.reshape(3, width).astype(np.int32)
    kv = PagedKV(3 * width, page, hkv, d, "fp4")
    cos, sin = backend.rope_table(width * page, d, THETA)
    cosn, sinn = cos.cpu().numpy(), sin.cpu().numpy()
    ws = backend.paged_workspace(kv, 3, hq)
    rows = {s: ([], []) for s in range(3)}

    def append(seqs, pos):
        n = len(seqs)
        q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (hq, hkv, hkv))
        q_out = torch.empty(n, hq, d, device="cuda")
        backend.dev_paged_append(kv, cuda(q), cuda(k), cuda(v), q_out, i32(pos), i32(table), cos, sin, seqs=i32(seqs))
        kr = values(*encode(rotate(k, cosn[pos], sinn[pos])))
        vr = values(*encode(v))
        for i, s in enumerate(seqs):
            rows[s][0].append(kr[i])
            rows[s][1].append(vr[i])
        return q_out

    append([s for s in range(3) for _ in range(lens[s])], [t for s in range(3) for t in range(lens[s])])
    for _ in range(6):
        q = append(range(3), lens)
        lens = [n + 1 for n in lens]
        out = torch.empty_like(q)
        backend.dev_paged_decode_attention(kv, q, i32(table), i32(lens), out, ws)
        qn, got = q.cpu().numpy(), out.cpu().numpy()
        for s in range(3):
            want, mag, size = attention(qn[s], np.array(rows[s][0]), np.array(rows[s][1]))
            assert (np.abs(got[s] - want) <= attention_bound(lens[s], d, mag, size)).all()
    back = [torch.zeros(3, hkv, max(lens), d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, i32(table), i32(lens), *back)
    for s in range(3):
        for i in range(2):
            assert same(back[i][s, :, :lens[s]].cpu().numpy().transpose(1, 0, 2), np.array(rows[s][i]))


@pytest.mark.parametrize("d", [128, 80])
def test_unaligned_pools(backend, d):
    """Pools at odd addresses take the other kernels, with the same results."""
    from bitnetrs_amd import PagedKV

    lens, page = [333, 20], 16
    pool = Pool4(rng_of("odd", d), lens, 2, d, page)

    def odd(x):
        t = torch.empty(x.size + 3, dtype=torch.uint8, device="cuda")[3:].view(x.shape)
        return t.copy_(cuda(x))

    kv = PagedKV.from_tensors(*(odd(x[n]) for x in (pool.codes, pool.exps) for n in "kv"))
    q = torch.randn(2, 6, d, device="cuda")
    out = torch.empty_like(q)
    backend.dev_paged_decode_attention(kv, q, i32(pool.table), i32(lens), out, backend.paged_workspace(kv, 2, 6))
    check_decode(pool, q.cpu().numpy(), out.cpu().numpy(), lens)
    back = [torch.zeros(2, 2, 333, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, i32(pool.table), i32(lens), *back)
    assert same(back[0][0].cpu().numpy().transpose(1, 0, 2), pool.rows("k", 0)[0])
    x = np.random.default_rng(3).standard_normal((333, 2, d)).astype(np.float32)
    backend.dev_paged_append(kv, None, cuda(x), cuda(x), None, i32(range(333)), i32(pool.table), seqs=i32([0] * 333))
    at = np.arange(333)
    check_rows(pool, kv, (pool.table[0, at // page], at % page), {"k": x, "v": x})


def test_offsets_past_32_bits(backend):
    """A page past 4 GiB of a pool: append, read and attention reach it."""
    from bitnetrs_amd import PagedKV

    d, page, hkv = 128, 64, 8
    n_pages = (5 << 30) // (hkv * page * d // 2)
    kv = PagedKV(n_pages, page, hkv, d, "fp4")
    rng = rng_of("far")
    x = rng.standard_normal((40, hkv, d)).astype(np.float32)
    table = i32([[n_pages - 1]])
    backend.dev_paged_append(kv, None, cuda(x), cuda(x * 2), None, i32(range(40)), table, seqs=i32([0] * 40))
    q = rng.standard_normal((1, hkv, d)).astype(np.float32)
    out = torch.empty(1, hkv, d, device="cuda")
    backend.dev_paged_decode_attention(kv, cuda(q), table, i32([40]), out, backend.paged_workspace(kv, 1, hkv))
    k, v = values(*encode(x)), values(*encode(x * 2))
    want, mag, size = attention(q[0], k, v)
    assert (np.abs(out[0].cpu().numpy() - want) <= attention_bound(40, d, mag, size)).all()
    back = [torch.zeros(1, hkv, 40, d, device="cuda") for _ in range(2)]
    backend.dev_paged_read(kv, table, i32([40]), *back)
    assert same(back[1][0].cpu().numpy().transpose(1, 0, 2), v)
    assert not kv.k[:-1].any()


def plant_infinity(pool, n, s, t, h, x, sign, exp, page):
    """Element x of a row as 6 * 2^(exp - 127), its group's others as zeros."""
    at = (pool.table[s, t // page], h, t % page)
    g = x // 32
    pool.exps[n][at][g] = exp
    pool.codes[n][at][16 * g: 16 * g + 16] = 0
    pool.codes[n][at][x // 2] = (15 if sign < 0 else 7) << 4 * (x % 2)


@pytest.mark.parametrize("hq", [4, 6, 8, 12])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (256, 16), (80, 32), (26, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_infinite_elements(backend, hq, d, page, wide):
    """Exponents 253 and 254 from elsewhere: a row of K whose score is -infinity is
    left out and one of +infinity makes the head NaN, however wide the table is; in
    V the columns show it, and nothing else."""
    lens = [200, 300, 150]
    pool = Pool4(rng_of("infinite", d), lens, 2, d, page, width=max(-(-300 // page), room(3, 2, page, wide)))
    plant_infinity(pool, "k", 0, 60, 1, d - 1, 1, 253, page)
    plant_infinity(pool, "k", 1, 299, 0, 3, -1, 254, page)
    plant_infinity(pool, "v", 2, 77, 1, d // 2, -1, 254, page)
    q, got = run_decode(backend, pool, hq, lens)
    G = hq // 2
    for s, row, h0, x, sign in ((0, 60, G, d - 1, 1), (1, 299, 0, 3, -1)):
        k, v = pool.rows("k", s)[0], pool.rows("v", s)[0]
        assert np.isinf(k[row]).sum() == 1
        nan = np.zeros(hq, bool)
        nan[h0:h0 + G] = q[s, h0:h0 + G, x] * sign > 0
        assert np.array_equal(np.isnan(got[s]), np.repeat(nan[:, None], d, 1)), s
        for h in np.nonzero(~nan)[0]:
            rows = np.arange(lens[s]) != (row if h // G == h0 // G else -1)
            want, mag, size = attention(q[s, h:h + 1], k[rows][:, [h // G]], v[rows][:, [h // G]])
            bound = attention_bound(int(rows.sum()), d, mag, size)
            assert (np.abs(got[s, h:h + 1] - want) <= bound).all(), (s, h)
    shows = np.zeros((hq, d), bool)
    shows[G:, d // 2] = True
    assert np.array_equal(~np.isfinite(got[2]), shows)
    v = pool.rows("v", 2)[0].copy()
    v[77, 1, d // 2] = 0
    want, mag, size = attention(q[2], pool.rows("k", 2)[0], v)
    bound = np.broadcast_to(attention_bound(150, d, mag, size), want.shape)
    assert (np.abs(got[2] - want) <= bound)[~shows].all()


@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (256, 16), (80, 32), (26, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_values_beside_non_finite_groups(backend, d, page, wide):
    """The heads and columns that no NaN group reaches have their values."""
    lens = [200, 200]
    pool = Pool4(rng_of("beside", d), lens, 2, d, page, width=max(-(-200 // page), room(2, 2, page, wide)))
    g = groups(d) - 1
    pool.exps["v"][pool.table[0, 77 // page], 1, 77 % page, g] = 255
    pool.exps["k"][pool.table[1, 150 // page], 0, 150 % page, 0] = 255
    q, got = run_decode(backend, pool, 6, lens)
    fine = np.ones((2, 6, d), bool)
    fine[0, 3:, 32 * g:] = False
    fine[1, :3] = False
    assert np.array_equal(np.isfinite(got), fine)
    for s in range(2):
        k, v = (np.nan_to_num(pool.rows(n, s)[0], nan=0.0) for n in "kv")
        want, mag, size = attention(q[s], k, v)
        off = np.abs(got[s] - want)
        assert (off <= attention_bound(200, d, mag, size))[fine[s]].all()
