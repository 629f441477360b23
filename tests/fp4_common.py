"""The paged cache's 4-bit rows in numpy, for their tests: 32 neighbouring
elements of a row share a power of two, codes are e2m1, two in a byte."""
from __future__ import annotations

import numpy as np
import torch

from paged_common import attention, attention_bound, i32, rotate  # noqa: F401  (for the tests)

GROUP = 32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float32)
TINY = np.float32(2.0 ** -100)


def groups(d):
    return -(-d // GROUP)


def encode(x):
    """Rows x [..., d] fp32 -> (codes uint8 [..., d/2], exponents uint8 [..., groups])."""
    x = np.asarray(x, np.float32)
    d, n = x.shape[-1], groups(x.shape[-1])
    y = np.zeros((*x.shape[:-1], n * GROUP), np.float32)
    y[..., :d] = x
    y = y.reshape(*x.shape[:-1], n, GROUP)
    fine = np.isfinite(y).all(-1)
    a = np.where(fine[..., None], np.abs(y), 0)
    m = np.maximum(a.max(-1), TINY).astype(np.float64)
    e = np.floor(np.log2(m / 3.5)).astype(np.int64)
    e = np.where(m >= 7 * 2.0 ** e, e + 1, np.where(m < 3.5 * 2.0 ** e, e - 1, e))  # where log2 rounded
    assert ((m >= 3.5 * 2.0 ** e) & (m < 7 * 2.0 ** e)).all()
    e = np.minimum(e, 125)
    z = a / 2.0 ** e[..., None]  # in 64 bits, exact
    # to the nearest of e2m1's values; between two of them to the one with the even code
    mid = (E2M1[1:] + E2M1[:-1]).astype(np.float64) / 2
    code = np.zeros(z.shape, np.uint8)
    for i, t in enumerate(mid):
        code += (z > t) | ((z == t) & ((i + 1) % 2 == 0))
    code = np.where(fine[..., None], code | np.signbit(y).astype(np.uint8) << 3, 0).astype(np.uint8)
    code = code.reshape(*x.shape[:-1], n * GROUP)[..., :d]
    exps = np.where(fine, e + 127, 255).astype(np.uint8)
    return (code[..., ::2] | code[..., 1::2] << 4).astype(np.uint8), exps


def values(codes, exps):
    """What codes [..., d/2] stand for, fp32 [..., d]."""
    codes, exps = np.asarray(codes), np.asarray(exps)
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    x = np.where(nib & 8, -E2M1[nib & 7], E2M1[nib & 7]).astype(np.float64)
    scale = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    with np.errstate(over="ignore"):
        return (x * np.repeat(scale, GROUP, -1)[..., : nib.shape[-1]]).astype(np.float32)


class Pool4:
    """A pool with random rows and its table; pages in no order, some unused."""

    def __init__(self, rng, lens, n_kv, d, page, width=None, spread=1.0):
        self.lens, self.page, self.n_kv, self.d = list(lens), page, n_kv, d
        width = width or max(1, -(-max(lens, default=1) // page))
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 2
        order = list(rng.permutation(n_pages))
        self.table = np.full((len(lens), width), -1, np.int32)
        for s, c in enumerate(need):
            self.table[s, :c] = [order.pop() for _ in range(c)]
        self.codes, self.exps = {}, {}
        for n in "kv":
            # each code and exponent as likely as another, so that all of a byte's 256 values are met
            self.codes[n] = rng.integers(0, 256, (n_pages, n_kv, page, d // 2)).astype(np.uint8)
            e = np.rint(125 + spread * rng.standard_normal((n_pages, n_kv, page, groups(d))))
            self.exps[n] = e.astype(np.uint8)

    def device(self):
        from bitnetrs_amd import PagedKV

        return PagedKV.from_tensors(*(torch.from_numpy(x[n]).cuda() for x in (self.codes, self.exps) for n in "kv"))

    def rows(self, n, s, length=None):
        """Values of rows 0..length-1 of sequence s, [length, n_kv, d], and
        which of them are there."""
        length = min(self.lens[s] if length is None else length, self.table.shape[1] * self.page)
        t = np.arange(max(length, 0))
        pages = self.table[s, t // self.page]
        there = (pages >= 0) & (pages < self.codes[n].shape[0])
        at = np.where(there, pages, 0)
        return values(self.codes[n][at, :, t % self.page], self.exps[n][at, :, t % self.page]), there


def same(a, b):
    """Equal bits, NaN for NaN."""
    a, b = np.ascontiguousarray(a, np.float32), np.ascontiguousarray(b, np.float32)
    both = np.isnan(a) & np.isnan(b)
    return np.array_equal(np.where(both, 0, a).view(np.uint32), np.where(both, 0, b).view(np.uint32))
