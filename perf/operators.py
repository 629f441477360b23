"""The paged key-value cache's operators as cases that can be timed and compared.

A paged cache holds the rows of many sequences in pages of one pool: codes [pages][kv heads][page rows][head dim],
kept in 32 bits ("f32"), bfloat16 ("bf16"), or 8 bits with one fp32 scale a row ("fp8": e4m3, "int8").  A table
[sequence][i] names the page that holds rows i * page .. (i + 1) * page - 1 of a sequence.  A case's "kind" says which
operator it is:

  append   HipBackend.dev_paged_append: q and k rotated at each token's own position, k and v quantised as they are
           written to their pages; then HipBackend.dev_paged_read of the rows just written, which gives the values
           that the codes stand for
  read     HipBackend.dev_paged_read: the rows of each sequence as fp32, in the layout that the prefill attention takes
  decode   HipBackend.dev_paged_decode_attention: one new token of each sequence over all rows of its own

`own` chooses between these calls and the same operators in elementary torch operations.  Head counts and the head
dimension of 20/5/128 are BitNet b1.58 2B's, the model that this library is configured for; the others are generic.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
THETA = 500000.0
TINY = 2.0 ** -100  # the least row maximum that a scale is made from
TOP = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "fp8": 1, "int8": 1}


def listed():
    return [
        # One token of one conversation: the smallest write there is, two launches' latency.
        {"name": "append_1_int8", "kind": "append", "format": "int8", "batch": 1, "lo": 900, "hi": 900, "new": 1,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # One token of each sequence of a full decode batch.
        {"name": "append_64_bf16", "kind": "append", "format": "bf16", "batch": 64, "lo": 64, "hi": 4000, "new": 1,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # Prompts of ragged lengths that continue cached conversations.
        {"name": "append_prompts_fp8", "kind": "append", "format": "fp8", "batch": 9, "lo": 1, "hi": 1900, "new": 1777,
         "heads": 32, "kv": 8, "d": 128, "page": 64},
        # A long document written into an empty cache.
        {"name": "append_document_int8", "kind": "append", "format": "int8", "batch": 1, "lo": 0, "hi": 0, "new": 4096,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # The cached part of one conversation, read back for a follow-up prompt's prefill.
        {"name": "read_700_bf16", "kind": "read", "format": "bf16", "batch": 1, "lo": 700, "hi": 700,
         "kv": 5, "d": 128, "page": 16},
        # The same for a full batch.
        {"name": "read_32_int8", "kind": "read", "format": "int8", "batch": 32, "lo": 100, "hi": 4096,
         "kv": 5, "d": 128, "page": 16},
        # A short chat turn: the smallest call, bound by latency.
        {"name": "decode_1_512_f32", "kind": "decode", "format": "f32", "batch": 1, "lo": 512, "hi": 512,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # One conversation at the end of the model's context.
        {"name": "decode_1_4096_bf16", "kind": "decode", "format": "bf16", "batch": 1, "lo": 4096, "hi": 4096,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # A full batch with lengths spread over the model's context.
        {"name": "decode_32_bf16", "kind": "decode", "format": "bf16", "batch": 32, "lo": 128, "hi": 4096,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # Odd sizes: 7 query heads a kv head, narrow heads, some sequences without a row.
        {"name": "decode_13_odd_int8", "kind": "decode", "format": "int8", "batch": 13, "lo": 1, "hi": 5001, "empty": 3,
         "heads": 14, "kv": 2, "d": 80, "page": 32},
        # One very long document: all of the card works on one sequence.
        {"name": "decode_1_131072_fp8", "kind": "decode", "format": "fp8", "batch": 1, "lo": 131072, "hi": 131072,
         "heads": 32, "kv": 8, "d": 128, "page": 64},
        # A large batch of long contexts, the largest work.
        {"name": "decode_64_long_int8", "kind": "decode", "format": "int8", "batch": 64, "lo": 1000, "hi": 32768,
         "heads": 20, "kv": 5, "d": 128, "page": 64},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, uniform in its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "decode", "decode"])
    heads, kv = rng.choice([(20, 5), (20, 5), (32, 8), (8, 8), (14, 2), (12, 1), (16, 8)])
    c = {"kind": kind, "format": rng.choice(["f32", "bf16", "fp8", "int8"]), "heads": heads, "kv": kv,
         "d": rng.choice([128, 128, 128, 64, 80, 96, 256]), "page": rng.choice([16, 16, 32, 64, 128])}
    row = kv * c["d"]
    if kind == "decode":
        c["batch"] = _spread(rng, 1, 64)
        # at most the longest listed sequence, and a fifth of the elements of the largest listed work
        top = max(2, min(131072, 128 * 1024 * 1024 // (row * c["batch"])))
        c["hi"] = _spread(rng, 1, top)
        c["lo"] = _spread(rng, 1, c["hi"])
        if c["batch"] > 3 and rng.random() < 0.3:
            c["empty"] = rng.randrange(1, c["batch"] // 2)
    elif kind == "read":
        c["batch"] = _spread(rng, 1, 32)
        c["hi"] = _spread(rng, 1, min(8192, max(2, 32 * 1024 * 1024 // (row * c["batch"]))))
        c["lo"] = _spread(rng, 1, c["hi"])
    else:
        c["batch"] = _spread(rng, 1, 64)
        c["new"] = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, min(4096, 8 * 1024 * 1024 // (row * c["batch"]))))
        c["hi"] = rng.randrange(0, 2000)
        c["lo"] = rng.randrange(0, c["hi"] + 1)
    return c


def _lens(case):
    """Rows of each sequence (before the new ones, where there are any): the first has the most, `empty` have none."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    n = [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]
    for i in range(case.get("empty", 0)):
        n[2 * i + 1] = 0
    return n


def _new(case):
    """New tokens of each sequence of an append: one each, or ragged with the first the longest."""
    rng = random.Random("%(batch)d %(new)d" % case)
    return [case["new"]] + [rng.randint(1, case["new"]) for _ in range(case["batch"] - 1)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    B, H, d, page, form = case["batch"], case["kv"], case["d"], case["page"], case["format"]
    lens = _lens(case)
    new = _new(case) if case["kind"] == "append" else [0] * B
    ends = [a + b for a, b in zip(lens, new)]
    wide = max(1, -(-max(ends) // page))  # pages that the table has room for, a sequence
    pages = sum(-(-n // page) for n in ends) + 3
    # Pages are handed out in no order, as a server that has run for a while has them.
    order = torch.randperm(pages, generator=g, device=DEV).cpu().tolist()
    rows = [[order.pop() if i * page < n else -1 for i in range(wide)] for n in ends]
    s = {"case": case, "table": torch.tensor(rows, dtype=torch.int32, device=DEV),
         "lens": torch.tensor(ends, dtype=torch.int32, device=DEV), "form": form, "page": page}

    def rows_like(*shape):
        # rows whose channels differ in size, as keys' do, and of one size as a whole
        return torch.randn(*shape, generator=g, device=DEV) * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))

    shape = (pages, H, page, d)
    for n in ("k", "v"):
        if form in TOP:
            x = rows_like(*shape).mul_(TOP[form] / 4).clamp_(-TOP[form], TOP[form])
            s[n] = (x.round_() if form == "int8" else x).to(DTYPE[form])
            s[n + "_scales"] = (0.7 + 0.6 * torch.rand(shape[:3], generator=g, device=DEV)) * (4 / TOP[form])
            del x
        else:
            s[n] = rows_like(*shape).to(DTYPE[form])
            s[n + "_scales"] = None
    if case["kind"] == "decode":
        s["q"] = torch.randn(B, case["heads"], d, generator=g, device=DEV)
        s["out"] = torch.zeros_like(s["q"])
        return s
    if case["kind"] == "append":
        T = sum(new)
        s["q"] = torch.randn(T, case["heads"], d, generator=g, device=DEV)
        s["new_k"], s["new_v"] = rows_like(T, H, d), rows_like(T, H, d)
        s["seqs"] = torch.tensor([b for b in range(B) for _ in range(new[b])], dtype=torch.int32, device=DEV)
        s["positions"] = torch.tensor([lens[b] + i for b in range(B) for i in range(new[b])], dtype=torch.int32, device=DEV)
        # the rotation's tables, which a program keeps: every position that a sequence can have
        i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
        angle = torch.arange(wide * page, dtype=torch.float64, device=DEV)[:, None] * THETA ** (-2 * i / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros_like(s["q"])
        s["starts"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        cap = max(new)
    else:
        s["starts"] = None
        cap = max(1, max(ends))
    s["k_out"], s["v_out"] = (torch.zeros(B, H, cap, d, device=DEV) for _ in range(2))
    return s


def run(s):
    return _own(s) if own else _plain(s)


@functools.lru_cache(None)
def _backend():
    """A program's one backend."""
    from bitnetrs_amd import HipBackend

    return HipBackend(0)


def _own(s):
    be, kind = _backend(), s["case"]["kind"]
    if "cache" not in s:  # what a program sets up once for a cache
        from bitnetrs_amd import PagedKV

        s["cache"] = PagedKV.from_tensors(s["k"], s["v"], s["k_scales"], s["v_scales"])
        if kind == "decode":
            s["workspace"] = be.paged_workspace(s["cache"], s["case"]["batch"], s["case"]["heads"])
    kv = s["cache"]
    if kind == "decode":
        be.dev_paged_decode_attention(kv, s["q"], s["table"], s["lens"], s["out"], s["workspace"])
        return s["out"]
    if kind == "append":
        be.dev_paged_append(kv, s["q"], s["new_k"], s["new_v"], s["q_out"], s["positions"], s["table"], s["cos"],
                            s["sin"], seqs=s["seqs"])
    be.dev_paged_read(kv, s["table"], s["lens"], s["k_out"], s["v_out"], starts=s["starts"])
    return (s["q_out"], s["k_out"], s["v_out"]) if kind == "append" else (s["k_out"], s["v_out"])


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "decode":
        return _attention(s)
    if kind == "append":
        s["q_out"].copy_(_rotated(s["q"], s))
        _write(s, "k", _rotated(s["new_k"], s))
        _write(s, "v", s["new_v"])
    for n in ("k", "v"):
        _rows_out(s, n)
    return (s["q_out"], s["k_out"], s["v_out"]) if kind == "append" else (s["k_out"], s["v_out"])


def _rotated(x, s):
    """Element i of the first half of a head turns with element i of the second."""
    at = s["positions"].long()
    c, n = s["cos"][at][:, None], s["sin"][at][:, None]
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * c - hi * n, hi * c + lo * n], -1)


def _write(s, n, x):
    """The new rows as codes (and scales) in their pages."""
    at, pool = s["positions"].long(), s[n]
    page, row = s["table"][s["seqs"].long(), at // s["page"]].long(), at % s["page"]
    if s["form"] in TOP:
        m = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
        top = torch.full_like(m, TOP[s["form"]])  # a tensor: by a number, torch multiplies with a rounded reciprocal
        code = x * (top / m)
        code = (code.round() if s["form"] == "int8" else code).to(pool.dtype)
        s[n + "_scales"][page, :, row] = (m / top)[..., 0]
        pool.view(torch.uint8)[page, :, row] = code.view(torch.uint8)
    else:
        pool[page, :, row] = x.to(pool.dtype)


def _values(s, n):
    """Every row that the table has room for, as fp32: [sequence][kv head][row][head dim]."""
    t = s["table"].clamp_min(0).long()
    pool = s[n]
    x = (pool.view(torch.uint8)[t].view(pool.dtype) if pool.dtype == DTYPE["fp8"] else pool[t]).float()
    if s["form"] in TOP:
        x = x * s[n + "_scales"][t][..., None]
    B, P, H, page, d = x.shape
    return x.transpose(1, 2).reshape(B, H, P * page, d)


def _rows_out(s, n):
    x, to = _values(s, n), s[n + "_out"]
    i = torch.arange(to.shape[2], device=DEV)
    first = torch.zeros_like(s["lens"]) if s["starts"] is None else s["starts"]
    at = first[:, None] + i
    there = (at < s["lens"][:, None])[:, None, :, None]
    at = at.clamp_max(x.shape[2] - 1).long()[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])
    to.copy_(torch.where(there, x.gather(2, at), to))


def _attention(s):
    k, v, q = _values(s, "k"), _values(s, "v"), s["q"]
    B, H, L, d = k.shape
    x = torch.matmul(q.view(B, H, -1, d), k.transpose(2, 3)) * (1 / math.sqrt(d))
    there = (torch.arange(L, device=DEV) < s["lens"][:, None])[:, None, None]
    x = torch.where(there, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(there.transpose(2, 3), v, 0.0)) / torch.where(total == 0, 1.0, total)
    return s["out"].copy_(out.view(q.shape))


def work(case):
    H, d, e = case["kv"], case["d"], BYTES[case["format"]]
    row = 2 * H * (d * e + (4 if e == 1 else 0))  # a token's codes and scales, k and v
    lens = _lens(case)
    if case["kind"] == "decode":
        n = sum(lens)
        return {"bytes": n * row + 8 * case["batch"] * case["heads"] * d, "flops": 4 * n * case["heads"] * d}
    if case["kind"] == "read":
        return {"bytes": sum(lens) * (row + 8 * H * d), "flops": sum(lens) * 2 * H * d}
    n = sum(_new(case))
    # the write (q, k, v in, q and the codes out), then the codes in and their values out
    return {"bytes": n * (8 * case["heads"] * d + 8 * H * d + row + row + 8 * H * d),
            "flops": n * (3 * (case["heads"] + H) * d + 6 * H * d)}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence, from the pages one by one."""
    s = prepare(case, seed)
    d, H, page, form = case["d"], case["kv"], case["page"], case["format"]
    table, ends = s["table"].cpu().tolist(), s["lens"].cpu().tolist()

    def rows(n, b, first, last):
        parts = []
        for i in range(first // page, -(-last // page)):
            x = s[n][table[b][i]].double()
            if form in TOP:
                x = x * s[n + "_scales"][table[b][i]].double()[:, :, None]
            parts.append(x)
        x = torch.cat(parts, 1)
        return x[:, first - first // page * page:][:, :last - first]

    if case["kind"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(ends):
            if n:
                q = s["q"][b].double().view(H, -1, d)
                x = (q[:, :, None] * rows("k", b, 0, n)[:, None]).sum(-1) if n < 4096 else q @ rows("k", b, 0, n).mT.contiguous()
                out[b] = (torch.softmax(x / d ** 0.5, -1) @ rows("v", b, 0, n)).reshape(-1, d)
        return out
    got = {n: s[n + "_out"].double() for n in ("k", "v")}
    if case["kind"] == "read":
        for b, n in enumerate(ends):
            for x in ("k", "v"):
                got[x][b, :, :n] = rows(x, b, 0, n)
        return got["k"], got["v"]

    def turned(x, step):
        # `step` rounds the products and their sums, where codes hang on it: that rounding is the definition's own
        at = s["positions"].long()
        c, n = s["cos"].double()[at][:, None], s["sin"].double()[at][:, None]
        lo, hi = x[..., : d // 2], x[..., d // 2:]
        return torch.cat([step(step(lo * c) - step(hi * n)), step(step(hi * c) + step(lo * n))], -1)

    def kept(x):
        # which code a value next to a border gets is defined in 32 bits; what the code stands for is computed in 64
        if form not in TOP:
            return x if form == "f32" else x.bfloat16().double()
        m = torch.clamp(x.abs().max(-1, keepdim=True).values, min=TINY)
        y = once(x * once(TOP[form] / m))
        return (torch.round(y) if form == "int8" else y.float().to(torch.float8_e4m3fn).double()) * m / TOP[form]

    def once(x):
        return x.float().double()

    def whole(x):
        return x

    new = {"k": kept(turned(s["new_k"].double(), whole if form == "f32" else once)), "v": kept(s["new_v"].double())}
    at = 0
    for b, n in enumerate(_new(case)):
        for x in ("k", "v"):
            got[x][b, :, :n] = new[x][at:at + n].transpose(0, 1)
        at += n
    return turned(s["q"].double(), whole), got["k"], got["v"]
