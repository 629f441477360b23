"""Paged pools whose attention is exact in fp32, so that one row too many or too
few shows however long the sequence is.

Each row has a bit and small whole numbers as values.  Its key is 4 in one place
where the bit is set and 0 elsewhere; a query is 12 sqrt(d) or -12 sqrt(d) there.
So the rows of a set bit (for a query below zero: the others) have one and the
same score, 48 above the rest, a weight of exactly 1, and the rest one of
exp(-48).  The sum of weights is then a count and the sum of values a whole
number, both below 2^24: exact in fp32 in any order.  A quotient of the two has
two roundings, of the reciprocal and of the product, 2^-24 each.  The other
rows' weights add at most n exp(-48) times 6.

What else rounds, by kernel:

- f32 rows on the matrix cores: nothing, a fp32 addition of such sums is exact but
  for the other rows' weights, which vanish in it.
- bf16, e4m3 and int8 rows there: one instruction adds 32 products and the sum so
  far, and keeps 2^-24 of the largest of them, cut downwards: 2 - exp(-48) comes out
  as 2 - 2^-22 beside a product of 4 (measured).  An instruction may so be off by
  2^-23 of the largest sum or value it meets; there are three for 32 rows (the
  parts of the weights), and one step of 32 rows more for each piece.  A wave
  adds the rows t with the same t / 32 mod 4 of a stretch of the sequence: the sum
  over such a stretch is at most twice the largest one from the start.  The sums
  of the 4 waves and of the pieces follow in fp32, at most 4 times as large.
- The kernel for other shapes (more than 16 query heads a kv head, pages that are no
  multiple of 16, other head dimensions) may take a score's factor 1 / sqrt(d) and
  the maximum in one rounding, while the maximum itself was rounded after the
  factor: the highest score's weight is then exp of that rounding's error, the same
  for all its rows, not 1.  It cancels in the quotient, but the sums are no longer
  whole numbers: each addition rounds, by 2^-24 of the sum at most, in the
  numerator and in the denominator, and each product of a weight and a value too.
  A wave adds 16 rows of each 64-row unit of its workgroup's share one after the
  other; then come the 4 waves, and the pieces or the groups of them and their
  members, fewer than the item's pieces in all."""
from __future__ import annotations

import numpy as np
import torch

from paged_common import DTYPE

# What the GPU tests run.  Two sequences of 256 kv heads of 16, 512 workgroups: shares of up to
# 8448 rows, so that a wave loads its list of 32 steps' pages three times over, cut
# anywhere; (page rows, pages that are not there).
LONG_SHAPE = ([8500, 8193], 256, 16)
LONG = [(16, 0), (48, 9), (64, 3), (128, 0)]
# Items of many workgroups: query heads, kv heads, head dim, page rows, lengths.
MANY = [(16, 1, 128, 16, [17, 21000]), (4, 1, 128, 64, [40000]), (12, 1, 80, 16, [30000]),
        (16, 1, 256, 16, [9000]), (14, 2, 128, 48, [12000, 1, 3000]), (20, 5, 128, 16, [4096] * 3),
        (20, 5, 128, 16, list(range(120, 200))), (17, 1, 64, 16, [9000]), (3, 1, 26, 16, [9000, 70]),
        (8, 4, 128, 5, [3000, 400]), (2, 1, 512, 8, [5000])]


class CountedPool:
    def __init__(self, seed, fmt, lens, hkv, d, page, missing=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda hi, *shape: torch.randint(0, hi, shape, generator=g, dtype=torch.int8)  # noqa: E731
        self.fmt, self.lens, self.hkv, self.d, self.page = fmt, list(lens), hkv, d, page
        width = -(-max(lens) // page)
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 1
        order = torch.randperm(n_pages, generator=g).tolist()
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for s, c in enumerate(need):
            self.table[s, :c] = torch.tensor([order.pop() for _ in range(c)], dtype=torch.int32)
        # pages that are not there, none of them a sequence's first or last
        for s, c in enumerate(need):
            for i in torch.randperm(max(c - 2, 0), generator=g)[:missing].tolist():
                self.table[s, 1 + i] = -1
        self.bits = rand(2, n_pages, hkv, page).bool()
        self.vals = 2 * (rand(7, n_pages, hkv, page, d) - 3)  # -6, -4 .. 6
        self.at = [7 * h % d for h in range(hkv)]
        self.scales = {"k": None, "v": None}
        if fmt in ("fp8", "int8"):  # codes times powers of two
            self.scales["k"] = torch.exp2(rand(3, n_pages, hkv, page).float())  # 1, 2, 4
            self.scales["v"] = torch.exp2(rand(3, n_pages, hkv, page).float() - 1)  # 1/2, 1, 2
        one = torch.ones(n_pages, hkv, page)
        kc = 4 * self.bits / (one if self.scales["k"] is None else self.scales["k"])
        k = torch.zeros(self.vals.shape, dtype=DTYPE[fmt])
        for h, x in enumerate(self.at):
            k[:, h, :, x] = kc[:, h].to(DTYPE[fmt])
        v = self.vals.float()
        if self.scales["v"] is not None:
            v /= self.scales["v"][..., None]
        self.codes = {"k": k, "v": v.to(DTYPE[fmt])}

    def device(self):
        from bitnetrs_amd import PagedKV

        sc = [None if self.scales[n] is None else self.scales[n].cuda() for n in "kv"]
        return PagedKV.from_tensors(self.codes["k"].cuda(), self.codes["v"].cuda(), *sc)

    def queries(self, hq):
        """One of each sign in turn, over the heads of a kv head and over kv heads."""
        g, size = hq // self.hkv, float(np.float32(12 * np.sqrt(self.d)))
        q = torch.zeros(len(self.lens), hq, self.d)
        for h in range(self.hkv):
            for j in range(g):
                q[:, h * g + j, self.at[h]] = size if (h + j) % 2 == 0 else -size
        return q

    def rows(self, s):
        """Bits [hkv, n] and values [hkv, n, d] of the rows of a sequence that are there,
        and their numbers."""
        t = torch.arange(self.lens[s])
        pages = self.table[s, t // self.page].long()
        t, pages = t[pages >= 0], pages[pages >= 0]
        return self.bits[pages, :, t % self.page].T, self.vals[pages, :, t % self.page].transpose(0, 1), t

    def expected(self, s, hq, weights=None):
        """What a kv head's queries above zero ([0]) and below it ([1]) get, in 64 bits,
        and how far a kernel may be off, both [2, hkv, d].  weights [n]: how often each
        row is counted (once)."""
        bits, vals, t = self.rows(s)
        v, w = vals.double(), torch.ones(len(t), dtype=torch.float64) if weights is None else weights.double()
        n, g, out, room = self.lens[s], hq // self.hkv, [], []
        matrix = g <= 16 and self.page % 16 == 0 and self.d % 16 == 0 and self.d <= 256
        for take in (bits, ~bits):
            p = take.double() * w
            none = p.sum(-1, keepdim=True) == 0  # no such row: all have the same score
            p = torch.where(none, w.expand_as(p), p)
            count = p.sum(-1, keepdim=True)
            x = torch.bmm(p[:, None], v)[:, 0] / count
            off = 6 * n * np.exp(-48.0)
            if matrix and self.fmt != "f32":
                pieces, largest = n // 128 + 1, 6.0
                for wave in range(4):
                    mine = (t // 32) % 4 == wave
                    if mine.any():
                        sums = (p[:, mine, None] * v[:, mine]).cumsum(1)
                        largest = max(largest, 2 * float(sums.abs().max()))
                off = off + (3 * (n / 32 + pieces) + 2 * (4 + pieces)) * 2.0 ** -23 * largest / count
            elif not matrix:
                share = -(-sum(-(-m // 64) for m in self.lens) * hq // 512)
                adds = 16 * share + 4 + n // 64 + 2
                off = off + 2 * (adds + 1) * 2.0 ** -24 * torch.bmm(p[:, None], v.abs())[:, 0] / count
            out.append(x)
            room.append(x.abs() * 2.0 ** -23 * (1 + 1e-6) + off)
        return torch.stack(out), torch.stack(room)
