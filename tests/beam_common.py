"""Page tables, beam selection and reordering in numpy, for their tests."""
from __future__ import annotations

import numpy as np


def pages_of(n, page):
    return -(-int(n) // page)


def extend(table, lens, new, free, count, page, n_tokens):
    """dev_paged_extend, sequence by sequence.  -> table, lens, count, seqs, positions, slots, offsets"""
    table, width = table.copy(), table.shape[1]
    count = min(max(int(count), 0), len(free))
    left, seqs, pos, slots, offsets = count, [], [], [], [0]
    out, stopped = [], False
    for s, (a, b) in enumerate(zip(lens, new)):
        a, b = max(int(a), 0), max(int(b), 0)
        if a + b > width * page:
            b = 0
        need = pages_of(a + b, page) - pages_of(a, page) if b else 0
        stopped = stopped or need > left or len(seqs) + b > n_tokens
        if not stopped:
            for i in range(need):
                left -= 1
                table[s, pages_of(a, page) + i] = free[left]
            for t in range(a, a + b):
                seqs.append(s)
                pos.append(t)
                p = int(table[s, t // page])
                slots.append(p * page + t % page if p >= 0 else -1)
            a += b
        out.append(a)
        offsets.append(len(seqs))
    pad = [-1] * (n_tokens - len(seqs))
    return table, out, left, seqs + pad, pos + pad, slots + pad, offsets


def release(table, lens, which, keep, free, count, page):
    """dev_paged_release.  -> table, lens, free, count"""
    table, free, width = table.copy(), free.copy(), table.shape[1]
    count = min(max(int(count), 0), len(free))
    out, stopped = [], False
    for s, n in enumerate(lens):
        n = max(int(n), 0)
        k = max(int(keep[s]), 0) if keep is not None else 0
        have = pages_of(min(n, width * page), page) - k if which[s] else 0
        stopped = stopped or count + max(have, 0) > len(free)
        if which[s] and not (stopped and have > 0):
            for i in range(max(have, 0)):
                free[count] = table[s, k + i]
                table[s, k + i] = -1
                count += 1
            n = min(n, k * page)
        out.append(n)
    return table, out, free, count


def select(logits, scores, k, done=None, eos=-1):
    """dev_beam_select in 64 bits.  -> tokens, parents, scores, done, and how far
    the scores of neighbours in the order are apart."""
    B, K, V = logits.shape
    tokens, parents = (np.zeros((B, k), np.int32) for _ in range(2))
    best, ended, gap = np.zeros((B, k)), np.zeros((B, k), np.uint8), np.inf
    for b in range(B):
        cand = []
        for j in range(K):
            x, base = logits[b, j].astype(np.float64), float(scores[b, j])
            if done is not None and done[b, j] and np.isfinite(base):
                rest = [t for t in range(k) if t != eos][: k - 1]
                cand += [(base, j, 0, eos)] + [(-np.inf, j, r + 1, t) for r, t in enumerate(rest)]
                continue
            with np.errstate(all="ignore"):
                lse = np.max(x) + np.log(np.exp(x - np.max(x)).sum())
            if not np.isfinite(base) or not np.isfinite(lse):
                cand += [(-np.inf, j, t, t) for t in range(k)]
                continue
            order = np.argsort(-x, kind="stable")[:k]
            cand += [(base + (x[t] - lse), j, r, int(t)) for r, t in enumerate(order)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for r, (y, j, _, t) in enumerate(cand[:k]):
            tokens[b, r], parents[b, r], best[b, r] = t, j, y
            ended[b, r] = bool(done is not None and done[b, j]) or t == eos
        for c, d in zip(cand[:k], cand[1: k + 1]):
            if c[1] != d[1] and np.isfinite(d[0]) and c[0] != d[0]:
                gap = min(gap, c[0] - d[0])
    return tokens, parents, best, ended, gap


def reorder(table, parents):
    """dev_beam_reorder.  -> table, src"""
    B, K = parents.shape
    out, src = np.empty_like(table), np.full(B * K, -1, np.int32)
    for b in range(B):
        par = [int(p) if 0 <= p < K else j for j, p in enumerate(parents[b])]
        ended = [i for i in range(K) if i not in par]
        first = {}
        for j, p in enumerate(par):
            if p not in first:
                first[p] = j
                row = p
            else:
                row = ended.pop(0)
                src[b * K + j] = b * K + first[p]
            out[b * K + j] = table[b * K + row]
        assert not ended
    return out, src
