"""The paged KV cache's definitions in numpy, for its tests: formats bit by
bit in 32-bit arithmetic, attention in 64 bits."""
from __future__ import annotations

import numpy as np
import torch

TINY = np.float32(2.0 ** -100)
TOP = {"int8": np.float32(127), "fp8": np.float32(448)}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn,
         "int8": torch.int8}
FORMATS = ("f32", "bf16", "fp8", "int8")


def rotate(x, cos, sin):
    """Half-split rotation, each product and sum rounded to fp32: x [n, h, d],
    cos / sin [n, d/2]."""
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    c, s = cos[:, None], sin[:, None]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1).astype(np.float32)


def encode(x, fmt):
    """Rows x [..., d] fp32 -> (codes as a torch tensor, scales or None)."""
    x = np.asarray(x, np.float32)
    if fmt in ("f32", "bf16"):
        return torch.from_numpy(x.copy()).to(DTYPE[fmt]), None
    fine = np.isfinite(x).all(-1, keepdims=True)
    m = np.maximum(np.abs(np.where(fine, x, 0)).max(-1, keepdims=True), TINY)
    y = np.where(fine, x, 0) * (TOP[fmt] / m)
    assert y.dtype == np.float32
    code = torch.from_numpy(np.rint(y) if fmt == "int8" else y).to(DTYPE[fmt])
    scale = np.where(fine, m / TOP[fmt], np.float32("nan")).astype(np.float32)
    return code, scale[..., 0]


def values(codes, scales):
    """What codes [..., d] stand for, fp32 [..., d]: one rounded product."""
    x = codes.float().numpy()
    return x if scales is None else (x * np.asarray(scales, np.float32)[..., None])


def attention(q, k, v):
    """softmax(q . k / sqrt(d)) v in 64 bits: q [H, d], k and v [n, Hkv, d];
    and the sum of weights times |v| that error bounds go by."""
    H, d = q.shape
    n, kv, _ = k.shape
    if n == 0:
        return np.zeros((H, d)), np.zeros((H, d)), np.zeros(H)
    g = H // kv
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    x = np.einsum("hgd,nhd->hgn", q.reshape(kv, g, d), k) / np.sqrt(d)
    size = np.einsum("hgd,nhd->hgn", np.abs(q).reshape(kv, g, d), np.abs(k)) / np.sqrt(d)
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out = np.einsum("hgn,nhd->hgd", p, v).reshape(H, d)
    return out, np.einsum("hgn,nhd->hgd", p, np.abs(v)).reshape(H, d), size.max(-1).reshape(H)


def attention_bound(n, d, mag, size):
    """How far fp32 arithmetic may be off, element by element.

    A score's dot product of d terms and its three factors: (d + 8) roundings
    of at most size = max sum |q k| / sqrt d; the exponential turns an error e
    of a score into 2 e at most of the weight (e << 1), its own error is under
    4 roundings; numerator and denominator both carry that.  Their sums run
    over at most n / 4 rows one after the other, and over at most 64 partial
    sums after that; the value of a row is a product, and the quotient one
    rounding.  mag = sum of weights times |v|.
    """
    eps = 2.0 ** -24
    score = (d + 8) * size[:, None] * eps
    return mag * (4 * score + 2 * (4 + n / 4 + 64 + 4) * eps) + 1e-37


class Pool:
    """A pool with random rows and its table; pages in no order, some unused."""

    def __init__(self, rng, fmt, lens, n_kv, d, page, width=None, spread=1.0):
        self.fmt, self.lens, self.page, self.n_kv, self.d = fmt, list(lens), page, n_kv, d
        width = width or max(1, -(-max(lens, default=1) // page))
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 2
        order = list(rng.permutation(n_pages))
        self.table = np.full((len(lens), width), -1, np.int32)
        for s, c in enumerate(need):
            self.table[s, :c] = [order.pop() for _ in range(c)]
        self.codes, self.scales = {}, {}
        for n in "kv":
            x = rng.standard_normal((n_pages, n_kv, page, d)).astype(np.float32)
            x *= np.exp(spread * rng.standard_normal((n_pages, n_kv, page, 1))).astype(np.float32)
            self.codes[n], self.scales[n] = encode(x, fmt)

    def device(self):
        from bitnetrs_amd import PagedKV

        sc = [None if self.scales[n] is None else torch.from_numpy(self.scales[n]).cuda()
              for n in "kv"]
        return PagedKV.from_tensors(self.codes["k"].cuda(), self.codes["v"].cuda(), *sc)

    def rows(self, n, s, length=None):
        """Values of rows 0..length-1 of sequence s, [length, n_kv, d], and
        which of them are there."""
        length = min(self.lens[s] if length is None else length, self.table.shape[1] * self.page)
        x = values(self.codes[n], self.scales[n])
        t = np.arange(max(length, 0))
        pages = self.table[s, t // self.page]
        there = (pages >= 0) & (pages < x.shape[0])
        return x[np.where(there, pages, 0), :, t % self.page], there


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")
