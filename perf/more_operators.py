"""Operators that serve many long conversations from a paged cache, as cases that can be timed and compared.

The paged cache itself (pages of one pool, a table that says which page holds which rows of a sequence) is described in
perf/operators.py.  A case's "kind" says which operator it is:

  append   HipBackend.dev_paged_append to a pool in 4 bits, then HipBackend.dev_paged_read of the rows just written.  32
           neighbouring elements of a row share a power of two, 2^e with 3.5 <= max|x| / 2^e < 7; a code is x / 2^e rounded
           to 0, 0.5, 1, 1.5, 2, 3, 4 or 6 and a sign (ties to the even code, 6 for all above 5)
  decode   HipBackend.dev_paged_decode_attention over a pool in 4 bits: one new token of each sequence over its rows
  rope     HipBackend.dev_rope: q and k, slices of one projection's output, rotated at each token's position, in pairs
           (i, i + dim/2) or (2i, 2i + 1) of the first `dim` elements of a head, by angles scaled for long contexts
  pages    HipBackend.dev_paged_extend: pages from a stack of free ones for each sequence's new tokens, the block table with
           them, and each new token's sequence, position and slot
  select   HipBackend.dev_beam_select: of each request's beams the best continuations over the whole vocabulary
  reorder  HipBackend.dev_beam_reorder and dev_paged_copy: the beams' tables follow the selection; where two beams go on
           from one, the second gets the pages of a beam that ended, with the rows copied that they do not share

`own` chooses between these calls and the same operators in elementary torch operations.  Head counts and the head
dimension of 20/5/128 and the vocabulary of 128256 are BitNet b1.58 2B's, the model that this library is configured for;
the others are generic.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
THETA = 500000.0
TINY = 2.0 ** -100  # the least maximum of a group that a power of two is made from
GROUP = 32
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # A long document written into an empty cache, 4 bits an element.
        {"name": "append_document", "kind": "append", "batch": 1, "lo": 0, "hi": 0, "new": 4096,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # One conversation at the end of the model's context: the smallest call, bound by latency.
        {"name": "decode_1_4096", "kind": "decode", "batch": 1, "lo": 4096, "hi": 4096,
         "heads": 20, "kv": 5, "d": 128, "page": 16},
        # A ragged batch of odd sizes: 7 query heads a kv head, narrow heads, some sequences without a row.
        {"name": "decode_29_odd", "kind": "decode", "batch": 29, "lo": 1, "hi": 6001, "empty": 3,
         "heads": 14, "kv": 2, "d": 80, "page": 32},
        # A large batch of long contexts, which is what 4 bits are for: the largest work.
        {"name": "decode_64_long", "kind": "decode", "batch": 64, "lo": 1000, "hi": 32768,
         "heads": 20, "kv": 5, "d": 128, "page": 64},
        # The new token of each sequence of a full decode batch, positions far behind the trained context.
        {"name": "rope_64_tokens", "kind": "rope", "type": "f32", "tokens": 64, "far": 131072, "heads": 20, "kv": 5,
         "d": 128, "dim": 128, "layout": "half", "scaling": "parts", "factor": 32.0},
        # The prompts of a batch in one call, a quarter of each head rotated in neighbouring pairs.
        {"name": "rope_prompts", "kind": "rope", "type": "bf16", "tokens": 16384, "far": 32768, "heads": 32, "kv": 8,
         "d": 128, "dim": 32, "layout": "interleaved", "scaling": "linear", "factor": 4.0},
        # A decode step's bookkeeping: one more token for each of 64 sequences.
        {"name": "pages_64_tokens", "kind": "pages", "batch": 64, "lo": 100, "hi": 4096, "new": 1, "page": 16},
        # Prompts of many sequences admitted at once, ragged, until the free pages run out.
        {"name": "pages_prompts", "kind": "pages", "batch": 300, "lo": 0, "hi": 2000, "new": 5000, "page": 16, "short": 0.9},
        # Four beams of one request.
        {"name": "select_1x4", "kind": "select", "batch": 1, "beams": 4, "vocab": 128256},
        # Eight beams of each request of a batch, some of which have ended.
        {"name": "select_16x8", "kind": "select", "batch": 16, "beams": 8, "vocab": 128256, "ended": 9},
        # The caches of four beams after 40 tokens of their own.
        {"name": "reorder_1x4", "kind": "reorder", "format": "bf16", "batch": 1, "beams": 4, "prompt": 700, "hi": 740,
         "kv": 5, "d": 128, "page": 16},
        # The same for a batch and long answers.
        {"name": "reorder_16x8", "kind": "reorder", "format": "bf16", "batch": 16, "beams": 8, "prompt": 300, "hi": 811,
         "kv": 5, "d": 128, "page": 16},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, uniform in its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "rope", "rope", "pages", "select", "reorder"])
    heads, kv = rng.choice([(20, 5), (20, 5), (32, 8), (8, 8), (14, 2), (12, 1), (16, 8)])
    d, page = rng.choice([128, 128, 128, 64, 80, 96, 256]), rng.choice([16, 16, 32, 64, 128])
    row = kv * d
    c = {"kind": kind}
    if kind == "append":
        batch = _spread(rng, 1, 64)
        c.update(batch=batch, heads=heads, kv=kv, d=d, page=page)
        c["new"] = 1 if rng.random() < 0.3 else _spread(rng, 2, max(2, min(4096, 2621440 // (row * batch))))
        c["hi"] = rng.randrange(0, 2000)
        c["lo"] = rng.randrange(0, c["hi"] + 1)
    elif kind == "decode":
        batch = _spread(rng, 1, 64)
        # a fifth of the elements of the largest listed work at most
        c.update(batch=batch, heads=heads, kv=kv, d=d, page=page,
                 hi=_spread(rng, 1, max(2, min(131072, 128 * 1024 * 1024 // (row * batch)))))
        c["lo"] = _spread(rng, 1, c["hi"])
        if batch > 3 and rng.random() < 0.3:
            c["empty"] = rng.randrange(1, batch // 2)
    elif kind == "rope":
        c.update(type=rng.choice(["f32", "bf16", "f16"]), tokens=_spread(rng, 1, 4096), far=_spread(rng, 100, 1 << 20),
                 heads=heads, kv=kv, d=d, dim=rng.choice([d, d, d // 2, d // 4]),
                 layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "parts"]),
                 factor=rng.choice([1.5, 4.0, 8.0, 32.0]))
    elif kind == "pages":
        c.update(batch=_spread(rng, 1, 1000), page=page, hi=rng.randrange(0, 4000))
        c["new"] = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, min(5000, 1000000 // c["batch"])))
        c["lo"] = rng.randrange(0, c["hi"] + 1)
        if rng.random() < 0.3:
            c["short"] = round(rng.uniform(0.3, 1.0), 2)
    elif kind == "select":
        c.update(batch=_spread(rng, 1, 32), beams=rng.randrange(1, 17), vocab=_spread(rng, 500, 128256))
        while c["batch"] * c["beams"] * c["vocab"] > 16 * 8 * 128256:
            c["batch"] //= 2
        if c["beams"] > 2 and rng.random() < 0.4:
            c["ended"] = rng.randrange(1, c["batch"] * c["beams"] // 2 + 1)
    else:
        c.update(format=rng.choice(["bf16", "f32"]), batch=_spread(rng, 1, 16), beams=rng.randrange(2, 17),
                 prompt=rng.randrange(0, 1000), kv=kv, d=d, page=page)
        most = 16 * 8 * 512 * 5 * 128 // (c["batch"] * c["beams"] * row * (2 if c["format"] == "f32" else 1))
        c["hi"] = c["prompt"] + _spread(rng, 1, max(2, min(2000, most)))
    return c


def _lens(case):
    """Rows of each sequence (before the new ones, where there are any): the first has the most, `empty` have none."""
    rng = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    n = [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]
    return [0 if i % 2 and i < 2 * case.get("empty", 0) else x for i, x in enumerate(n)]


def _new(case):
    """New tokens of each sequence: one each, or ragged with the first the longest."""
    rng = random.Random("%(batch)d %(new)d" % case)
    return [case["new"]] + [rng.randint(1, case["new"]) for _ in range(case["batch"] - 1)]


def _rates(case):
    """Radians a position of each pair, and what the rotated values are multiplied with."""
    dim, s, kind = case["dim"], case["factor"], case["scaling"]
    base = THETA * s ** (dim / (dim - 2)) if kind == "ntk" else THETA
    rates = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if kind == "linear":
        rates = [r / s for r in rates]
    if kind == "parts":  # by how often a pair turns over the 4096 positions of the training: 1 stretched, 32 as it was
        keep = [min(max((4096 * r / (2 * math.pi) - 1) / 31, 0.0), 1.0) for r in rates]
        rates = [r * (k + (1 - k) / s) for r, k in zip(rates, keep)]
    return rates, 0.1 * math.log(s) + 1 if kind == "parts" else 1.0


def _parents(case):
    """Which beam each one of a reorder goes on from: some twice or more, some not at all."""
    rng = random.Random("%(batch)d %(beams)d %(hi)d" % case)
    return [[min(rng.randrange(case["beams"]), rng.randrange(case["beams"])) for _ in range(case["beams"])]
            for _ in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    made = {"append": _cache, "decode": _cache, "rope": _tokens, "pages": _stack, "select": _logits, "reorder": _beams}
    s = made[case["kind"]](case, g)
    s["case"] = case
    return s


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows_like(g, *shape):
    """Rows whose channels differ in size, as keys' do."""
    return _normal(g, *shape) * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))


def _table(ends, page, g, spare=3):
    """Pages for so many rows of each sequence, in no order, as a server that has run for a while has them."""
    wide = max(1, -(-max(ends) // page))
    counts = [-(-n // page) for n in ends]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device=DEV).cpu().tolist()
    return _i32([[order.pop() if i < n else -1 for i in range(wide)] for n in counts]), pages


def _cache(case, g):
    B, H, d, page = case["batch"], case["kv"], case["d"], case["page"]
    lens = _lens(case)
    new = _new(case) if case["kind"] == "append" else [0] * B
    ends = [a + b for a, b in zip(lens, new)]
    table, pages = _table(ends, page, g)
    s = {"table": table, "lens": _i32(ends), "page": page}
    # codes of rows of one size, two to a byte, and their groups' powers of two with it
    shape = (pages, H, page, -(-d // GROUP))
    s.update({n: torch.randint(0, 256, (pages, H, page, d // 2), generator=g, device=DEV, dtype=torch.uint8) for n in "kv"})
    s.update({n + "_scales": torch.randint(124, 128, shape, generator=g, device=DEV, dtype=torch.uint8) for n in "kv"})
    if case["kind"] == "decode":
        s["q"] = _normal(g, B, case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
        return s
    T = sum(new)
    s["q"] = _normal(g, T, case["heads"], d)
    s["new_k"], s["new_v"] = _rows_like(g, T, H, d), _rows_like(g, T, H, d)
    s["seqs"] = _i32([b for b in range(B) for _ in range(new[b])])
    s["positions"] = _i32([lens[b] + i for b in range(B) for i in range(new[b])])
    # the rotation's tables, which a program keeps: every position that a sequence can have
    i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
    angle = torch.arange(table.shape[1] * page, dtype=torch.float64, device=DEV)[:, None] * THETA ** (-2 * i / d)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_out"] = torch.zeros_like(s["q"])
    s["starts"] = _i32(lens)
    s["k_out"], s["v_out"] = (torch.zeros(B, H, max(new), d, device=DEV) for _ in range(2))
    return s


def _tokens(case, g):
    n, H, kv, d = case["tokens"], case["heads"], case["kv"], case["d"]
    x = _normal(g, n, (H + 2 * kv) * d).to(DTYPE[case["type"]])  # q, k and v of a token side by side
    s = {"q": x[:, :H * d].view(n, H, d), "k": x[:, H * d:(H + kv) * d].view(n, kv, d)}
    s["positions"] = torch.randint(0, case["far"], (n,), generator=g, device=DEV, dtype=torch.int32)
    s["q_out"], s["k_out"] = (torch.zeros(n, h, d, dtype=x.dtype, device=DEV) for h in (H, kv))
    return s


def _stack(case, g):
    B, page = case["batch"], case["page"]
    lens, new = _lens(case), _new(case)
    wide = -(-(max(lens) + case["new"]) // page) + 1
    have = [-(-n // page) for n in lens]
    more = sum(-(-(a + b) // page) - h for a, b, h in zip(lens, new, have))
    free = max(1, int(more * case.get("short", 1.2)))
    order = torch.randperm(sum(have) + free, generator=g, device=DEV).to(torch.int32)
    where = torch.arange(wide, device=DEV) < _i32(have)[:, None]
    table = torch.full((B, wide), -1, dtype=torch.int32, device=DEV)
    table[where] = order[free:]
    T = sum(new)
    s = {"table": table, "lens": _i32(lens), "new": _i32(new), "free": order[:free].clone(), "count": _i32([free])}
    s.update({n: torch.zeros(T, dtype=torch.int32, device=DEV) for n in ("seqs", "positions")})
    s["slots"] = torch.zeros(T, dtype=torch.int64, device=DEV)
    s["offsets"] = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    s["lens_out"], s["count_out"] = torch.zeros_like(s["lens"]), torch.zeros_like(s["count"])
    return s


def _logits(case, g):
    B, K, V = case["batch"], case["beams"], case["vocab"]
    s = {"logits": 2.5 * _normal(g, B, K, V), "scores": -5 * torch.rand(B, K, generator=g, device=DEV)}
    ended = torch.arange(B * K, device=DEV).view(B, K) * 7 % (B * K) < case.get("ended", 0)
    s["done"] = ended.to(torch.uint8)
    s["eos"] = V - 1
    s["tokens"], s["parents"] = (torch.zeros(B, K, dtype=torch.int32, device=DEV) for _ in range(2))
    s["scores_out"], s["done_out"] = torch.zeros_like(s["scores"]), torch.zeros_like(s["done"])
    return s


def _beams(case, g):
    B, K, page, n = case["batch"], case["beams"], case["page"], case["hi"]
    shared = case["prompt"] // page  # full pages of the prompt, the same for a request's beams
    wide = -(-n // page)
    pages = B * (shared + K * (wide - shared)) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    prompt = order[:B * shared].view(B, 1, shared).expand(B, K, shared)
    rest = order[B * shared:B * (shared + K * (wide - shared))].view(B, K, wide - shared)
    s = {"table": torch.cat([prompt, rest], 2).reshape(B * K, wide).contiguous(), "page": page}
    shape = (pages, case["kv"], page, case["d"])
    s["k"], s["v"] = (_normal(g, *shape).to(DTYPE[case["format"]]) for _ in range(2))
    s["parents"] = _i32(_parents(case))
    s["starts"] = _i32([shared * page] * (B * K))
    s["lens"] = _i32([n] * (B * K))
    s["table_out"] = torch.zeros_like(s["table"])
    s["src"] = torch.zeros(B * K, dtype=torch.int32, device=DEV)
    return s


def run(s):
    return _own(s) if own else _plain(s)


@functools.lru_cache(None)
def _backend():
    """A program's one backend."""
    from bitnetrs_amd import HipBackend

    return HipBackend(0)


def _own(s):
    be, c = _backend(), s["case"]
    kind = c["kind"]
    if "kept" not in s:  # what a program sets up once
        from bitnetrs_amd import PagedKV, Rope

        if kind in ("append", "decode"):
            s["kept"] = PagedKV.from_tensors(s["k"], s["v"], s["k_scales"], s["v_scales"])
        elif kind == "reorder":
            s["kept"] = PagedKV.from_tensors(s["k"], s["v"])
        elif kind == "rope":
            scaled = {} if c["scaling"] == "none" else {"scaling": c["scaling"], "factor": c["factor"]}
            if c["scaling"] == "parts":
                scaled.update(original=4096, magnitude=0.1 * math.log(c["factor"]) + 1)
            s["kept"] = Rope(c["dim"], THETA, layout=c["layout"], **scaled)
        else:
            s["kept"] = None
        if kind == "decode":
            s["workspace"] = be.paged_workspace(s["kept"], c["batch"], c["heads"])
        if kind == "select":
            s["workspace"] = be.beam_workspace(c["batch"], c["beams"], c["vocab"], c["beams"])
    kept = s["kept"]
    if kind == "decode":
        be.dev_paged_decode_attention(kept, s["q"], s["table"], s["lens"], s["out"], s["workspace"])
    elif kind == "append":
        be.dev_paged_append(kept, s["q"], s["new_k"], s["new_v"], s["q_out"], s["positions"], s["table"], s["cos"],
                            s["sin"], seqs=s["seqs"])
        be.dev_paged_read(kept, s["table"], s["lens"], s["k_out"], s["v_out"], starts=s["starts"])
    elif kind == "rope":
        be.dev_rope(kept, s["q"], s["k"], s["positions"], s["q_out"], s["k_out"])
    elif kind == "pages":
        be.dev_paged_extend(s["table"], s["lens"], s["new"], s["free"], s["count"], c["page"], s["seqs"], s["positions"],
                            s["offsets"], s["lens_out"], s["count_out"], slots=s["slots"])
    elif kind == "select":
        be.dev_beam_select(s["logits"], s["scores"], s["tokens"], s["parents"], s["scores_out"], s["workspace"],
                           done=s["done"], eos=s["eos"], done_out=s["done_out"])
    else:
        be.dev_beam_reorder(s["table"], s["parents"], s["table_out"], s["src"])
        be.dev_paged_copy(kept, s["table_out"], s["src"], s["lens"], starts=s["starts"])
    return _outputs(s)


def _outputs(s):
    names = {"append": ("q_out", "k_out", "v_out"), "decode": ("out",), "rope": ("q_out", "k_out"),
             "pages": ("table", "lens_out", "count_out", "seqs", "positions", "slots", "offsets"),
             "select": ("tokens", "parents", "scores_out", "done_out"), "reorder": ("table_out", "src", "k", "v")}
    return {n: s[n] for n in names[s["case"]["kind"]]}


def _plain(s):
    {"append": _append, "decode": _attention, "rope": _rope, "pages": _extend, "select": _select,
     "reorder": _reorder}[s["case"]["kind"]](s)
    return _outputs(s)


def _append(s):
    at = s["positions"].long()
    c, n = s["cos"][at][:, None], s["sin"][at][:, None]
    s["q_out"].copy_(_halves(s["q"], c, n))
    _write(s, "k", _halves(s["new_k"], c, n))
    _write(s, "v", s["new_v"])
    _rows_out(s, "k")
    _rows_out(s, "v")


def _halves(x, c, n):
    """Element i of the first half of a head turns with element i of the second."""
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * c - hi * n, hi * c + lo * n], -1)


def _write(s, n, x):
    """The new rows as codes and powers of two in their pages."""
    T, H, d = x.shape
    full = -(-d // GROUP)
    y = torch.zeros(T, H, full * GROUP, device=DEV)
    y[..., :d] = x
    y = y.view(T, H, full, GROUP)
    m = y.abs().amax(-1, keepdim=True).clamp_min(TINY)
    e = (m.view(torch.int32) + 0x200000 >> 23) - 129  # 3.5 * 2^e <= m < 7 * 2^e
    a = y.abs() * torch.exp2(-e.float())
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + 8 * torch.signbit(y)).view(T, H, -1)[..., :d]
    at = s["positions"].long()
    page, row = s["table"][s["seqs"].long(), at // s["page"]].long(), at % s["page"]
    s[n][page, :, row] = (code[..., ::2] + 16 * code[..., 1::2]).byte()
    s[n + "_scales"][page, :, row] = (e[..., 0] + 127).byte()


def _values(s, n):
    """Every row that the table has room for, as fp32: [sequence][kv head][row][head dim]."""
    t = s["table"].clamp_min(0).long()
    x = s[n][t].long()
    B, P, H, page, half = x.shape
    known = torch.tensor(E2M1 + [-v for v in E2M1], device=DEV)
    x = torch.stack([known[x % 16], known[x // 16]], -1).view(B, P, H, page, 2 * half)
    e = torch.exp2(s[n + "_scales"][t].float() - 127).repeat_interleave(GROUP, -1)[..., :2 * half]
    return (x * e).transpose(1, 2).reshape(B, H, P * page, 2 * half)


def _rows_out(s, n):
    x, to = _values(s, n), s[n + "_out"]
    at = s["starts"][:, None] + torch.arange(to.shape[2], device=DEV)
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
    s["out"].copy_(out.view(q.shape))


def _rope(s):
    rates, size = _rates(s["case"])
    # in 64 bits: a float has no place left for the angle of a far position
    angle = s["positions"].double()[:, None, None] * torch.tensor(rates, dtype=torch.float64, device=DEV)
    c, n = (angle.cos() * size).float(), (angle.sin() * size).float()
    s["q_out"].copy_(_turned(s["q"].float(), c, n, s["case"]))
    s["k_out"].copy_(_turned(s["k"].float(), c, n, s["case"]))


def _turned(x, c, n, case):
    dim = case["dim"]
    if case["layout"] == "half":
        first = _halves(x[..., :dim], c, n)
    else:
        lo, hi = x[..., 0:dim:2], x[..., 1:dim:2]
        first = torch.stack([lo * c - hi * n, hi * c + lo * n], -1).flatten(-2)
    return torch.cat([first, x[..., dim:]], -1)


def _extend(s):
    page, table, T = s["case"]["page"], s["table"], s["seqs"].numel()
    B, wide = table.shape
    lens, new = s["lens"].long().clamp_min(0), s["new"].long().clamp_min(0)
    have = (lens + page - 1) // page
    new = torch.where(lens + new <= wide * page, new, 0)
    need = (lens + new + page - 1) // page - have
    free = s["count"].long().clamp(0, s["free"].numel())
    # in order, up to the first sequence that does not fit
    fits = (need.cumsum(0) <= free) & (new.cumsum(0) <= T)
    new, need = torch.where(fits, new, 0), torch.where(fits, need, 0)
    ends, pages = new.cumsum(0), need.cumsum(0)
    i = torch.arange(wide, device=DEV) - have[:, None]
    taken = free - 1 - ((pages - need)[:, None] + i)
    table.copy_(torch.where((i >= 0) & (i < need[:, None]), s["free"][taken.clamp(0, s["free"].numel() - 1)], table))
    s["offsets"][1:] = ends
    s["lens_out"].copy_(lens + new)
    s["count_out"].copy_(free - pages[-1:])
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(ends, t, right=True)
    there, seq = seq < B, seq.clamp_max(B - 1)
    at = torch.where(there, lens[seq] + t - (ends - new)[seq], 0)
    slot = table[seq, at // page].long() * page + at % page
    s["seqs"].copy_(torch.where(there, seq, -1))
    s["positions"].copy_(torch.where(there, at, -1))
    s["slots"].copy_(torch.where(there, slot, -1))


def _select(s):
    x, base, done = s["logits"], s["scores"].double(), s["done"].bool()
    B, K, V = x.shape
    # a beam's own best: by their logits, then the lowest index, as whole numbers that are all different
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)
    key = order * (1 << 32) - torch.arange(V, device=DEV)
    best = (-key.topk(K, -1).values) % (1 << 32)
    # the sum in 64 bits: beams that are near each other change places otherwise
    m = x.amax(-1, keepdim=True).double()
    z = (m + torch.exp(x.double() - m).sum(-1, keepdim=True).log())
    y = base[..., None] + (x.gather(-1, best).double() - z)
    # a beam that has ended goes on with the end's token alone, at its score
    rank = torch.arange(K, device=DEV)
    ends = torch.where(rank == 0, base[..., None], -math.inf)
    y = torch.where(done[..., None], ends, y).view(B, K * K)
    best = torch.where(done[..., None], torch.where(rank == 0, s["eos"], rank - 1), best).view(B, K * K)
    top = y.sort(dim=-1, descending=True, stable=True)
    at = top.indices[:, :K]
    s["scores_out"].copy_(top.values[:, :K])
    s["tokens"].copy_(best.gather(1, at))
    s["parents"].copy_(at // K)
    s["done_out"].copy_(done.gather(1, at // K) | (s["tokens"] == s["eos"]))


def _reorder(s):
    table, parents, page = s["table"], s["parents"].long(), s["page"]
    B, K = parents.shape
    j = torch.arange(K, device=DEV)
    same = parents[:, :, None] == parents[:, None, :]
    heir = ~(same & (j < j[:, None])).any(2)  # the first that goes on from its parent has the parent's pages
    first = (same * (K - j)).argmax(2)
    live = (parents[:, :, None] == j).any(1)
    ended = live.int().sort(dim=1, stable=True).indices  # the others those of the beams that ended, in order
    extra = (~heir).long().cumsum(1) - 1
    row = torch.where(heir, parents, ended.gather(1, extra.clamp_min(0)))
    base = torch.arange(B, device=DEV)[:, None] * K
    s["table_out"].copy_(table[(base + row).view(-1)])
    s["src"].copy_(torch.where(heir, -1, base + first).view(-1))
    # the rows that such a beam does not share
    src, at = s["src"].long(), torch.arange(table.shape[1] * page, device=DEV)
    rows = (src >= 0)[:, None] & (at >= s["starts"][:, None]) & (at < s["lens"][:, None])
    b, t = rows.nonzero(as_tuple=True)
    to, of = s["table_out"][b, t // page].long(), s["table_out"][src[b], t // page].long()
    s["k"][to, :, t % page] = s["k"][of, :, t % page]
    s["v"][to, :, t % page] = s["v"][of, :, t % page]


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + case["kv"])
        return {"bytes": 2 * n * case["d"] * SIZE[case["type"]] + 4 * case["tokens"], "flops": 3 * n * case["dim"]}
    if kind == "pages":
        n, t = sum(_new(case)), case["batch"]
        return {"bytes": 16 * n + 16 * t + 8 * (n // case["page"]), "flops": 0}
    if kind == "select":
        n = case["batch"] * case["beams"] - case.get("ended", 0)
        return {"bytes": 4 * n * case["vocab"] + 16 * case["batch"] * case["beams"], "flops": 4 * n * case["vocab"]}
    if kind == "reorder":
        wide, extra = -(-case["hi"] // case["page"]), sum(case["beams"] - len(set(p)) for p in _parents(case))
        rows = case["hi"] - case["prompt"] // case["page"] * case["page"]
        return {"bytes": 8 * case["batch"] * case["beams"] * wide
                + 4 * extra * rows * case["kv"] * case["d"] * SIZE[case["format"]], "flops": 0}
    H, d = case["kv"], case["d"]
    row = 2 * H * (d // 2 + -(-d // GROUP))  # a token's codes and powers of two, k and v
    lens = _lens(case)
    if kind == "decode":
        return {"bytes": sum(lens) * row + 8 * case["batch"] * case["heads"] * d, "flops": 4 * sum(lens) * case["heads"] * d}
    n = sum(_new(case))
    # the write (q, k, v in, q and the codes out), then the codes in and their values out
    return {"bytes": n * (8 * case["heads"] * d + 8 * H * d + row + row + 8 * H * d),
            "flops": n * (3 * (case["heads"] + H) * d + 6 * H * d)}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence; whole numbers have none, nor have rows that are copied."""
    kind = case["kind"]
    if kind in ("pages", "reorder"):
        return None
    s = prepare(case, seed)
    if kind == "rope":
        rates, size = _rates(case)
        got = {}
        for n in ("q", "k"):
            x = s[n].double()
            y = x.clone()
            for i, r in enumerate(rates):
                a, b = (i, i + case["dim"] // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
                angle = (s["positions"].double() * r)[:, None]
                y[..., a] = size * (x[..., a] * angle.cos() - x[..., b] * angle.sin())
                y[..., b] = size * (x[..., b] * angle.cos() + x[..., a] * angle.sin())
            got[n + "_out"] = y
        return got
    if kind == "select":
        B, K, V = s["logits"].shape
        best = torch.empty(B, K, dtype=torch.float64, device=DEV)
        for b in range(B):
            y = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
            for k in s["done"][b].nonzero()[:, 0].tolist():
                y[k] = -math.inf
                y[k, s["eos"]] = s["scores"][b, k].double()
            best[b] = y.flatten().sort(descending=True).values[:K]
        return {"tokens": None, "parents": None, "scores_out": best, "done_out": None}
    d, H, page = case["d"], case["kv"], case["page"]
    table, ends = s["table"].cpu().tolist(), s["lens"].cpu().tolist()
    known = torch.tensor([v * sign for sign in (1, -1) for v in E2M1], dtype=torch.float64, device=DEV)

    def rows(n, b, count):
        at = torch.tensor(table[b][:-(-count // page)], device=DEV)
        codes = s[n][at]
        x = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=DEV)
        x[..., 0::2], x[..., 1::2] = known[(codes & 15).long()], known[(codes >> 4).long()]
        e = s[n + "_scales"][at].double() - 127
        x *= 2.0 ** e[..., torch.arange(d, device=DEV) // GROUP]
        return x.transpose(0, 1).reshape(H, -1, d)[:, :count]

    if kind == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(ends):
            if n:
                q = s["q"][b].double().view(H, -1, d)
                x = q @ rows("k", b, n).mT.contiguous()
                out[b] = (torch.softmax(x / d ** 0.5, -1) @ rows("v", b, n)).reshape(-1, d)
        return {"out": out}

    def once(x):
        return x.float().double()

    def turned(x, step):
        # `step` rounds the products and their sums, where codes hang on it: that rounding is the definition's own
        at = s["positions"].long()
        c, n = s["cos"].double()[at][:, None], s["sin"].double()[at][:, None]
        lo, hi = x[..., : d // 2], x[..., d // 2:]
        return torch.cat([step(step(lo * c) - step(hi * n)), step(step(hi * c) + step(lo * n))], -1)

    def kept(x):
        out = torch.empty_like(x)
        for i in range(0, d, GROUP):
            part = x[..., i:i + GROUP]
            m = part.abs().max(-1, keepdim=True).values.clamp(min=TINY)
            unit = 2.0 ** torch.floor(torch.log2(m / 3.5))
            unit = torch.where(m >= 7 * unit, 2 * unit, torch.where(m < 3.5 * unit, unit / 2, unit))
            a = (part / unit).abs()
            step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
            out[..., i:i + GROUP] = torch.sign(part) * (torch.round(a / step) * step).clamp(max=6) * unit
        return out

    got = {"q_out": turned(s["q"].double(), lambda x: x), "k_out": s["k_out"].double(), "v_out": s["v_out"].double()}
    new = {"k_out": kept(turned(s["new_k"].double(), once)), "v_out": kept(s["new_v"].double())}
    at = 0
    for b, n in enumerate(_new(case)):
        for x in new:
            got[x][b, :, :n] = new[x][at:at + n].transpose(0, 1)
        at += n
    return got
