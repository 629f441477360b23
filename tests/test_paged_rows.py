"""The pools of tests/paged_rows.py on the CPU: the weights are what they are said
to be, and a row left out, counted twice or taken for another shows."""
import numpy as np
import pytest
import torch

from paged_common import attention, values
from paged_rows import LONG, LONG_SHAPE, MANY, CountedPool

# As on the GPU; of the long sequences 4 of the kv heads.
SHAPES = [(s[0], *s, 2) for s in MANY] + [(page, 8, 4, LONG_SHAPE[2], page, LONG_SHAPE[0], m) for page, m in LONG]


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("seed,hq,hkv,d,page,lens,missing", SHAPES)
def test_one_row_shows(fmt, seed, hq, hkv, d, page, lens, missing):
    """Leaving out or doubling any one row that a query weighs moves some output by
    more than twice what the kernel may be off by."""
    pool = CountedPool(seed, fmt, lens, hkv, d, page, missing)
    for s in range(len(lens)):
        bits, vals, t = pool.rows(s)
        if len(t) < 2:
            continue
        want, room = pool.expected(s, hq)
        for side, take in enumerate((bits, ~bits)):
            count = take.sum(-1)[:, None, None]
            # the mean without row t: it moves by (mean - v) / (count - 1); with it twice, by (v - mean) / (count + 1)
            moved = (vals.double() - want[side][:, None]).abs() / (count + 1)
            far = (moved > 2 * room[side][:, None]).any(-1)
            assert far[take].all(), (s, side)
    # and by doing it, for a few rows: at the ends and in the middle
    n = pool.rows(0)[0].shape[1]
    want, room = pool.expected(0, hq)
    for t in {0, n // 3, n - 1}:
        for times in (0, 2):
            w = torch.ones(n)
            w[t] = times
            got, _ = pool.expected(0, hq, w)
            assert ((got - want).abs() > room).any(-1).any(0).all(), (t, times)


@pytest.mark.parametrize("fmt", ["f32", "bf16", "fp8", "int8"])
def test_expected_is_attention(fmt):
    """The counts and means are softmax attention, in 64 bits, over what the codes
    stand for."""
    pool = CountedPool(3, fmt, [300, 1, 77], 3, 32, 16, 1)
    q = pool.queries(12).numpy()
    for s, n in enumerate(pool.lens):
        t = np.arange(n)
        pages = pool.table.numpy()[s, t // 16]
        t, pages = t[pages >= 0], pages[pages >= 0]
        k, v = (values(pool.codes[x], pool.scales[x])[pages, :, t % 16] for x in "kv")
        ref = attention(q[s], k, v)[0].reshape(3, 4, 32)
        want, room = pool.expected(s, 12)
        for h in range(3):
            for j in range(4):
                side = (h + j) % 2
                # both in 64 bits: sums of at most 300 values of at most 6
                off = room[side, h].numpy() + 300 * 6 * 2.0 ** -53
                assert (np.abs(ref[h, j] - want[side, h].numpy()) <= off).all()


def test_sums_are_exact_in_fp32():
    """Values and counts stay whole numbers below 2^24, scales powers of two, and
    every format holds its codes."""
    assert 6 * max(max(s[4]) for s in MANY) < 2 ** 24 and 6 * max(LONG_SHAPE[0]) < 2 ** 24
    for fmt in ("f32", "bf16", "fp8", "int8"):
        pool = CountedPool(5, fmt, [200], 2, 16, 16)
        assert (values(pool.codes["v"], pool.scales["v"]) == pool.vals.numpy()).all()
        key = values(pool.codes["k"], pool.scales["k"])
        assert (key.sum(-1) == 4 * pool.bits.numpy()).all() and (np.abs(key) <= 4).all()
