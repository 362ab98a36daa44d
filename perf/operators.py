"""What the speed of the text decoder's operators is measured on: the calls that a program which
writes a line's or a page's text token by token makes, through this library's public entry points.

Four kinds of pass: a step's queries, keys and values normed, rotated and written into the paged
cache, and the cache read back ("kv"); attention over a prompt of packed documents ("attn");
attention of single tokens over the cache ("decode"); a step of beam search with the reordering of
the beams' pages ("beam").

With `own` the passes are the library's calls, queued on its context's stream; otherwise the same
results from elementary torch operations. `exact` evaluates the definitions in float64.
"""
from __future__ import annotations

import functools
import math
import os
import random
import sys

import torch

own = False
GPU = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
QMAX = {"i8": 127.0, "e4m3": 448.0}
EPS, TINY = 1e-6, 1e-30


def listed():
    return [
        # One text line's next token: the smallest model's step, latency alone.
        {"name": "kv_line_step", "kind": "kv", "seqs": 1, "new": 1, "past": 200, "hq": 8, "hk": 8, "d": 64, "rot": 64,
         "theta": 1e4, "pairs": "halves", "page": 16, "type": "f16", "cache": "f16"},
        # The next token of every beam of a page's 36 lines, four beams a line.
        {"name": "kv_beams_step", "kind": "kv", "seqs": 144, "new": 1, "past": 300, "hq": 16, "hk": 4, "d": 128, "rot": 64,
         "theta": 1e4, "pairs": "adjacent", "page": 16, "type": "bf16", "cache": "i8"},
        # Prompts of long documents: eight ragged ones, about 32 000 tokens.
        {"name": "kv_prompts", "kind": "kv", "seqs": 8, "new": 4096, "past": 0, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "theta": 5e5, "pairs": "halves", "page": 64, "type": "bf16", "cache": "e4m3"},
        # One line's image tokens (109 steps, the PP recogniser's neck on a wide line), all seen by all.
        {"name": "attn_line", "kind": "attn", "docs": 1, "most": 109, "prefix": 1.0, "hq": 8, "hk": 8, "d": 64, "cap": 0.0,
         "slopes": False, "pad": 0, "type": "f16"},
        # A page's 36 lines packed into one row: image tokens as prefix, the text so far after them.
        {"name": "attn_lines", "kind": "attn", "docs": 36, "most": 130, "prefix": 0.7, "hq": 16, "hk": 4, "d": 64, "cap": 0.0,
         "slopes": True, "pad": 37, "type": "bf16"},
        # A whole page: some 2000 image tokens as prefix and 900 of text; capped scores.
        {"name": "attn_page", "kind": "attn", "docs": 1, "most": 2929, "prefix": 0.7, "hq": 16, "hk": 4, "d": 128, "cap": 50.0,
         "slopes": False, "pad": 0, "type": "bf16"},
        # Long documents, causal but for a short prefix.
        {"name": "attn_long", "kind": "attn", "docs": 2, "most": 5000, "prefix": 0.1, "hq": 32, "hk": 8, "d": 128, "cap": 0.0,
         "slopes": False, "pad": 0, "type": "bf16"},
        # One line's next token, over its own 16-bit cache.
        {"name": "decode_line", "kind": "decode", "seqs": 1, "len": 201, "hq": 8, "hk": 8, "d": 64, "cap": 0.0, "slopes": False,
         "page": 16, "type": "f16", "cache": "f16"},
        # The beams of a page's lines, distance bias and capped scores.
        {"name": "decode_beams", "kind": "decode", "seqs": 144, "len": 700, "hq": 16, "hk": 4, "d": 128, "cap": 30.0,
         "slopes": True, "page": 16, "type": "bf16", "cache": "i8"},
        # A few very long documents: the cache's bandwidth.
        {"name": "decode_long", "kind": "decode", "seqs": 4, "len": 131072, "hq": 32, "hk": 8, "d": 128, "cap": 0.0,
         "slopes": False, "page": 64, "type": "bf16", "cache": "e4m3"},
        # One line, four beams, the ocrs alphabet (97 classes).
        {"name": "beam_line", "kind": "beam", "groups": 1, "beams": 4, "vocab": 97, "first": False, "len": 60, "hk": 4, "d": 64,
         "page": 16, "type": "f32", "cache": "f16"},
        # 64 lines, eight beams each, a large vocabulary.
        {"name": "beam_large", "kind": "beam", "groups": 64, "beams": 8, "vocab": 128000, "first": False, "len": 500, "hk": 4,
         "d": 128, "page": 64, "type": "bf16", "cache": "bf16"},
    ]


def draw(rng):
    """A case of the same ranges: sizes spread over their logarithm, odd ones among them, none that
    costs more than the largest listed one of its kind."""
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    def heads():
        hk = rng.choice([1, 2, 4, 8])
        return {"hk": hk, "hq": hk * rng.choice([1, 2, 3, 4, 8]), "d": rng.choice([32, 64, 64, 80, 96, 128, 128])}

    kind = rng.choice(["kv", "attn", "decode", "beam"])
    page, t16 = rng.choice([16, 32, 64]), rng.choice(["f16", "bf16"])
    if kind == "kv":
        c = {"kind": kind, **heads(), "theta": rng.choice([1e4, 5e5]), "pairs": rng.choice(["halves", "adjacent"]), "page": page,
             "type": t16, "cache": rng.choice([t16, "i8", "e4m3"])}
        c["rot"] = rng.choice([c["d"], c["d"], 32, 0])
        if rng.random() < 0.4:  # a step of single tokens
            n = log(1, 200)
            c.update(seqs=n, new=1, past=log(1, min(2000, 60000 // n)))
        else:
            c.update(seqs=log(1, 8), new=log(2, 1100), past=rng.choice([0, 0, log(1, 300)]))
        return c
    if kind == "attn":
        docs, h = log(1, 40), heads()
        most = int(min(7000, (2.3e11 / (4 * h["hq"] * h["d"])) ** 0.5)) // docs
        return {"kind": kind, "docs": docs, "most": log(1, most), "prefix": rng.choice([0.0, 0.1, 0.5, 0.7, 1.0]), **h, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.4, "pad": rng.choice([0, 0, log(1, 99)]),
                "type": t16}
    if kind == "decode":
        n = log(1, 200)
        return {"kind": kind, "seqs": n, "len": log(1, min(100000, 230000 // n)), **heads(), "cap": rng.choice([0.0, 0.0, 30.0]),
                "slopes": rng.random() < 0.4, "page": page, "type": t16, "cache": rng.choice([t16, "i8", "e4m3"])}
    n, w = log(1, 64), rng.choice([1, 2, 3, 4, 5, 8])
    t = rng.choice(["f32", t16])
    return {"kind": kind, "groups": n, "beams": w, "vocab": log(50, 50000 if t == "f32" else 100000), "first": rng.random() < 0.2, "len": log(1, 500),
            "hk": rng.choice([1, 2, 4]), "d": rng.choice([32, 64, 128]), "page": page,
            "type": t, "cache": t16}


# ---- sizes that follow from a case --------------------------------------------------------------
def _counts(n, most, salt):
    """n ragged lengths: the first the most, the others between a quarter of it and all of it."""
    rng = random.Random(n * 1000003 + most * 31 + salt)
    return [most] + [rng.randint(max(1, most // 4), most) for _ in range(n - 1)]


def _kv_sizes(c):
    past = _counts(c["seqs"], c["past"], 1) if c["past"] else [0] * c["seqs"]
    return past, _counts(c["seqs"], c["new"], 2)


# ---- inputs --------------------------------------------------------------------------------------
def _cache(gen, c, pages, filled=True):
    """A paged cache's memory, [pages][heads][page][dim] and a scale a vector for the 8-bit ones."""
    shape = (pages, c["hk"], c["page"], c["d"])
    out = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device=GPU, dtype=torch.float16)
        s = None
        if c["cache"] == "i8":
            x = (x * 40).round().clamp(-127, 127).to(torch.int8)
        elif c["cache"] == "e4m3":
            x = (x.float() * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            x = x.to(TYPES[c["cache"]])
        if c["cache"] in QMAX:
            s = (0.6 + torch.rand(shape[:3], generator=gen, device=GPU)) * (0.025 if c["cache"] == "i8" else 0.009)
        out[name], out[name + "_scale"] = x if filled else torch.zeros_like(x), s if filled or s is None else torch.zeros_like(s)
    return out


def _tables(gen, lens, page, spare=0):
    """Every sequence's pages, anywhere in the pool (-1 past its last), and how many pages that takes."""
    need = [-(-n // page) for n in lens]
    total, width = sum(need), max(max(need), 1)
    perm = torch.randperm(total, generator=gen, device=GPU).to(torch.int32)
    col = torch.arange(width, device=GPU)[None]
    n = torch.tensor(need, device=GPU)[:, None]
    first = torch.cumsum(n, 0) - n
    at = (first + col).clamp(max=max(total - 1, 0))
    table = torch.where(col < n, perm[at] if total else torch.zeros_like(at, dtype=torch.int32), -1).to(torch.int32)
    return table.contiguous(), total + spare


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(GPU).manual_seed(int(seed) * 7919 + 17)
    rn = lambda *shape: torch.randn(*shape, generator=gen, device=GPU)  # noqa: E731
    s = {"case": c}
    kind = c["kind"]
    i32 = dict(dtype=torch.int32, device=GPU)
    t = TYPES[c["type"]]
    if kind == "kv":
        past, new = _kv_sizes(c)
        lens = [p + n for p, n in zip(past, new)]
        s["table"], pages = _tables(gen, lens, c["page"])
        s["cache"] = _cache(gen, c, pages)
        n, width = sum(new), (c["hq"] + 2 * c["hk"]) * c["d"]
        # Projections of normed activations: channels of unlike size.
        s["qkv"] = (rn(n, width) * (0.3 + rn(1, width).abs())).to(t)
        s["seq"] = torch.repeat_interleave(torch.arange(len(new), device=GPU), torch.tensor(new, device=GPU)).to(torch.int32)
        s["pos"] = torch.cat([torch.arange(p, p + k, **i32) for p, k in zip(past, new)])
        s["lens"] = torch.tensor(lens, **i32)
        s["q_norm"], s["k_norm"] = 1 + 0.2 * rn(c["d"]), 1 + 0.2 * rn(c["d"])
        s["q"] = torch.empty(n, c["hq"], c["d"], dtype=t, device=GPU)
        s["k_out"] = torch.empty(len(new), max(lens), c["hk"], c["d"], dtype=t, device=GPU)
        s["v_out"] = torch.empty_like(s["k_out"])
    elif kind == "attn":
        lens = _counts(c["docs"], c["most"], 3)
        n = sum(lens) + c["pad"]
        s["q"], s["k"], s["v"] = ((rn(n, h, c["d"]) * a).to(t) for h, a in ((c["hq"], 1.5), (c["hk"], 1.0), (c["hk"], 1.0)))
        off = [0]
        for k in lens:
            off.append(off[-1] + k)
        s["docs"] = torch.tensor(off, **i32)
        s["prefix"] = torch.tensor([int(k * c["prefix"]) for k in lens], **i32)
        s["slopes"] = _slopes(c)
        s["out"] = torch.empty_like(s["q"])
    elif kind == "decode":
        lens = _counts(c["seqs"], c["len"], 4)
        s["table"], pages = _tables(gen, lens, c["page"])
        s["cache"] = _cache(gen, c, pages)
        s["lens"] = torch.tensor(lens, **i32)
        s["q"] = (rn(c["seqs"], c["hq"], c["d"]) * 1.5).to(t)
        s["slopes"] = _slopes(c)
        s["out"] = torch.empty_like(s["q"])
    else:
        g, w, v = c["groups"], c["beams"], c["vocab"]
        # A confident reader's logits: a few tokens stand out of the many.
        x = rn(g * w, v) * 2
        top = torch.randint(0, v, (g * w, 6), generator=gen, device=GPU)
        s["logits"] = x.scatter_(1, top, 9 + 3 * rn(g * w, 6)).to(t)
        s["scores"] = -30 * torch.rand(g, w, generator=gen, device=GPU)
        s["finished"] = (torch.rand(g, w, generator=gen, device=GPU) < 0.15).to(torch.int32)
        s["eos"] = min(2, v - 1)
        if c["first"]:  # the first step: one beam a group holds the start, the others nothing
            s["scores"][:, 0], s["scores"][:, 1:] = 0, -math.inf
            s["finished"].zero_()
        lens = [n for n in _counts(g, c["len"], 5) for _ in range(w)]
        s["table"], pages = _tables(gen, lens, c["page"], g * w)
        s["cache"] = _cache(gen, c, pages)
        s["spare"] = torch.arange(pages - g * w, pages, **i32)  # a page a beam, none of the sequences'
        for name in ("k", "v"):
            s["cache"][name][pages - g * w:] = 0
        s["lens"] = torch.tensor(lens, **i32)
        s["o_scores"] = torch.empty(g, w, device=GPU)
        s["o_parents"], s["o_tokens"], s["o_finished"] = (torch.empty(g, w, **i32) for _ in range(3))
        s["o_table"], s["o_lens"], s["o_used"] = torch.empty_like(s["table"]), torch.empty_like(s["lens"]), torch.empty_like(s["lens"])
    return s


def _slopes(c):
    """Distance slopes in a geometric row, one a head."""
    if not c["slopes"]:
        return None
    return 2.0 ** (-8.0 * (1 + torch.arange(c["hq"], device=GPU, dtype=torch.float32)) / c["hq"])


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"kv": _plain_kv, "attn": _plain_attn, "decode": _plain_decode, "beam": _plain_beam}[s["case"]["kind"]](s)


@functools.lru_cache(None)
def _library():
    """The library and the context that a program keeps."""
    sys.path.insert(0, os.path.join(os.getcwd(), "wgpu-ocr_amd"))
    import ocrhip
    return ocrhip, ocrhip.Context()


def _handle(s):
    """The cache's handle over the caller's memory, kept as long as that."""
    if "handle" not in s:
        ocrhip, ctx = _library()
        m = s["cache"]
        pages, heads, page, dim = m["k"].shape
        s["handle"] = ocrhip.KvCache(ctx, pages, page, heads, dim, s["case"]["cache"],
                                     memory=(m["k"], m["v"], m["k_scale"], m["v_scale"]))
    return s["handle"]


def _run_own(s):
    ocrhip, ctx = _library()
    c = s["case"]
    kind = c["kind"]
    if kind == "kv":
        cache = _handle(s)
        cache.append(s["table"], s["seq"], s["pos"], s["qkv"], s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, rot=c["rot"],
                     theta=c["theta"], pairs=c["pairs"])
        cache.read(s["table"], s["lens"], s["k_out"], s["v_out"])
        return {"q": s["q"], "k": s["k_out"], "v": s["v_out"]}
    if kind == "attn":
        ocrhip.attention(ctx, s["q"], s["k"], s["v"], s["out"], s["docs"], prefix=s["prefix"], scale=c["d"] ** -0.5, cap=c["cap"],
                         slopes=s["slopes"])
        return s["out"]
    if kind == "decode":
        _handle(s).attend(s["table"], s["lens"], s["q"], s["out"], scale=c["d"] ** -0.5, cap=c["cap"], slopes=s["slopes"])
        return s["out"]
    ocrhip.beam_select(ctx, s["logits"], s["scores"], s["finished"], s["eos"], s["o_scores"], s["o_parents"], s["o_tokens"],
                       s["o_finished"])
    _handle(s).fork(s["table"], s["lens"], s["o_parents"], s["spare"], s["o_table"], s["o_lens"], s["o_used"])
    return _beam_outputs(s, s["o_scores"], s["o_parents"], s["o_tokens"], s["o_finished"], s["o_table"], s["o_lens"], s["o_used"])


def _beam_outputs(s, scores, parents, tokens, finished, table, lens, used):
    first = s["cache"]["k"].shape[0] - s["spare"].numel()
    return {"scores": scores, "parents": parents, "tokens": tokens, "finished": finished, "table": table, "lens": lens, "used": used,
            "k_spare": s["cache"]["k"][first:], "v_spare": s["cache"]["v"][first:]}


# ---- the plain forms -----------------------------------------------------------------------------
def _rotate(x, pos, c):
    """x [n][heads][d] float32 with its first `rot` values rotated; the angles in float64."""
    r = c["rot"]
    if r == 0:
        return x
    freq = c["theta"] ** (-torch.arange(0, r, 2, device=GPU, dtype=torch.float64) / r)
    angle = (pos.double()[:, None] * freq)[:, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    y = x.clone()
    if c["pairs"] == "halves":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y[..., : r // 2], y[..., r // 2: r] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _write(cache, name, page, row, x, fmt):
    """The vectors x [n][heads][d] float32 at (page, row), in the cache's form."""
    if fmt not in QMAX:
        cache[name][page, :, row] = x.to(TYPES[fmt])
        return
    amax = x.abs().amax(-1)
    keep = amax > TINY
    y = x * torch.where(keep, QMAX[fmt] / amax, 0)[..., None]
    code = y.round().to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn).view(torch.uint8)
    cache[name][page, :, row] = code
    cache[name + "_scale"][page, :, row] = torch.where(keep, amax / QMAX[fmt], 0)


def _values(cache, name, fmt, table):
    """The vectors of every sequence's pages, float32 [sequences][positions][heads][d]."""
    x = cache[name][table.clamp(min=0).long()]
    x = (x.view(torch.float8_e4m3fn) if fmt == "e4m3" else x).float()
    if fmt in QMAX:
        x = x * cache[name + "_scale"][table.clamp(min=0).long()][..., None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_kv(s):
    c, m = s["case"], s["cache"]
    n, hq, hk, d, t = s["qkv"].shape[0], c["hq"], c["hk"], c["d"], TYPES[c["type"]]
    q, k, v = s["qkv"].float().view(n, hq + 2 * hk, d).split([hq, hk, hk], 1)
    q = _rotate(_norm(q, s["q_norm"]), s["pos"], c).to(t)
    k = _rotate(_norm(k, s["k_norm"]), s["pos"], c)
    pos = s["pos"].long()
    page, row = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    _write(m, "k", page, row, k, c["cache"])
    _write(m, "v", page, row, v, c["cache"])
    most = s["k_out"].shape[1]
    there = torch.arange(most, device=GPU)[None] < s["lens"][:, None]
    out = [torch.where(there[..., None, None], _values(m, x, c["cache"], s["table"])[:, :most], 0).to(t) for x in ("k", "v")]
    return {"q": q, "k": out[0], "v": out[1]}


def _softmax_rows(x, seen):
    """exp(x - max) and its sums over the last axis, nothing where not seen; rows that see nothing weigh nothing."""
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0, top))
    return e, e.sum(-1, keepdim=True)


def _cap(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _plain_attn(s):
    c = s["case"]
    n, hk, d, g = s["q"].shape[0], c["hk"], c["d"], c["hq"] // c["hk"]
    q = s["q"].float().view(n, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * n, d)
    k, v = (s[x].float().transpose(0, 1).contiguous() for x in ("k", "v"))
    x = torch.matmul(q, k.transpose(1, 2).contiguous()).view(hk, g, n, n) * d ** -0.5
    x = _cap(x, c["cap"])
    at = torch.arange(n, device=GPU)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(hk, g, 1, 1) * (at[:, None] - at[None]).abs()
    doc = torch.searchsorted(s["docs"], at.int(), right=True) - 1
    inside = doc < c["docs"]
    start, pre = s["docs"][:-1][doc.clamp(max=c["docs"] - 1)], s["prefix"][doc.clamp(max=c["docs"] - 1)]
    seen = (doc[:, None] == doc[None]) & inside[:, None] & ((at[None] <= at[:, None]) | (at[None] < (start + pre)[:, None]))
    e, total = _softmax_rows(x, seen)
    del x
    o = torch.matmul(e.view(hk, g * n, n), v).view(hk, g, n, d) / torch.where(total > 0, total, 1)
    return o.permute(2, 0, 1, 3).reshape(n, c["hq"], d).to(TYPES[c["type"]])


def _plain_decode(s):
    c, m = s["case"], s["cache"]
    n, hk, d, g = c["seqs"], c["hk"], c["d"], c["hq"] // c["hk"]
    k, v = (_values(m, x, c["cache"], s["table"]).transpose(1, 2).contiguous() for x in ("k", "v"))
    q = s["q"].float().view(n, hk, g, d)
    x = _cap(torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5, c["cap"])
    at = torch.arange(k.shape[2], device=GPU)[None, None, None]
    last = s["lens"].view(n, 1, 1, 1) - 1
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hk, g, 1) * (last - at)
    e, total = _softmax_rows(x, at <= last)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1)
    return o.reshape(n, c["hq"], d).to(TYPES[c["type"]])


def _plain_beam(s):
    c, m = s["case"], s["cache"]
    g, w, v, page = c["groups"], c["beams"], c["vocab"], c["page"]
    x = s["logits"].double()  # a float32 sum of many would decide between neighbours
    x = x - torch.logsumexp(x, 1, keepdim=True)
    over = s["finished"].view(-1, 1) != 0
    x = torch.where(over, torch.where(torch.arange(v, device=GPU)[None] == s["eos"], 0.0, -math.inf), x)
    x = (x + s["scores"].double().view(-1, 1)).view(g, w * v)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    best, at = best[:, :w].float(), at[:, :w]
    parents, tokens = at // v, at % v
    finished = (s["finished"].gather(1, parents) != 0) | (tokens == s["eos"])
    rows = (parents + torch.arange(g, device=GPU)[:, None] * w).view(-1)
    lens = s["lens"][rows]
    full, tail = lens // page, lens % page
    # The first child of a parent keeps its part-filled page, the others get a copy.
    earlier = torch.ones(w, w, dtype=torch.bool, device=GPU).tril(-1)
    first = ~((parents[:, :, None] == parents[:, None]) & earlier).any(2).view(-1)
    used = (tail > 0) & ~first
    col = torch.arange(s["table"].shape[1], device=GPU)[None]
    table = torch.where(col < (full + (tail > 0))[:, None], s["table"][rows], -1)
    source = table.gather(1, full.long().clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    table = torch.where((col == full[:, None]) & used[:, None], s["spare"][:, None], table)
    copied = (used[:, None] & (torch.arange(page, device=GPU)[None] < tail[:, None]))[:, None, :, None]
    for name in ("k", "v"):
        here = m[name][s["spare"].long()]
        m[name][s["spare"].long()] = torch.where(copied, m[name][source.long().clamp(min=0)], here)
    i = torch.int32
    return _beam_outputs(s, best, parents.to(i), tokens.to(i), finished.to(i), table.to(i), lens.to(i), used.to(i))


# ---- the work ------------------------------------------------------------------------------------
def _bytes_of(fmt):
    return 1 if fmt in QMAX else 2


def work(case):
    c, kind = case, case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
    held = c["d"] * _bytes_of(c["cache"]) + (4 if c["cache"] in QMAX else 0) if "cache" in c else 0  # bytes of a vector
    if kind == "kv":
        past, new = _kv_sizes(c)
        n, total = sum(new), sum(past) + sum(new)
        values = n * (c["hq"] + 2 * c["hk"]) * c["d"]
        there = len(new) * max(p + k for p, k in zip(past, new))
        # The projections in, q out, the new vectors written, every vector read back, K and V whole.
        return {"bytes": values * size + n * c["hq"] * c["d"] * size + 2 * c["hk"] * held * (n + total) + 2 * there * c["hk"] * c["d"] * size,
                "flops": 10 * values}
    if kind == "attn":
        lens = _counts(c["docs"], c["most"], 3)
        pairs = 0
        for k in lens:
            p = int(k * c["prefix"])
            pairs += p * p + (k * (k + 1) - p * (p + 1)) // 2  # prefix rows see the prefix, the others their past
        n = sum(lens) + c["pad"]
        return {"bytes": n * 2 * (c["hq"] + c["hk"]) * c["d"] * size, "flops": 4 * pairs * c["hq"] * c["d"]}
    if kind == "decode":
        total = sum(_counts(c["seqs"], c["len"], 4))
        return {"bytes": total * 2 * c["hk"] * held + 2 * c["seqs"] * c["hq"] * c["d"] * size, "flops": 4 * total * c["hq"] * c["d"]}
    rows = c["groups"] * c["beams"]
    width = -(-c["len"] // c["page"])
    # The logits once; the tables in and out. How many tails are copied depends on the values: about half of them.
    return {"bytes": rows * (c["vocab"] * size + 8 * width + 40) + rows * c["page"] * c["hk"] * held,
            "flops": 3 * rows * c["vocab"]}


# ---- the definitions in float64 ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"kv": _exact_kv, "attn": _exact_attn, "decode": _exact_decode, "beam": _exact_beam}[case["kind"]](case, s)


def _e4m3(y):
    """Values in [-448, 448] to the nearest of 1 + 3 mantissa bits, ties to even, subnormal under 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_held(x, fmt):
    """What the cache holds of a float64 vector, as the value it stands for."""
    if fmt not in QMAX:
        return x.to(TYPES[fmt]).double()
    scale = x.abs().amax(-1, keepdim=True) / QMAX[fmt]
    y = x / torch.where(scale > 0, scale, 1.0)
    return (torch.round(y) if fmt == "i8" else _e4m3(y)) * scale


def _exact_sequences(s, c, name):
    """One float64 [positions][heads][d] a sequence, from the pages as they are."""
    out = []
    for row, n in zip(s["table"].tolist(), s["lens"].tolist()):
        pages = torch.tensor(row[: -(-n // c["page"])], device=GPU, dtype=torch.int64)
        x = s["cache"][name][pages]
        x = (x.view(torch.float8_e4m3fn).float() if c["cache"] == "e4m3" else x).double()
        if c["cache"] in QMAX:
            x = x * s["cache"][name + "_scale"][pages].double().unsqueeze(-1)
        out.append(torch.cat(list(x.transpose(1, 2)), 0)[:n] if n else x.new_zeros(0, c["hk"], c["d"]))
    return out


def _exact_kv(c, s):
    x = s["qkv"].double().reshape(-1, c["hq"] + 2 * c["hk"], c["d"])
    heads = torch.arange(x.shape[1], device=GPU)
    weight = torch.ones(x.shape[1], c["d"], dtype=torch.float64, device=GPU)
    weight[: c["hq"]], weight[c["hq"]: c["hq"] + c["hk"]] = s["q_norm"].double(), s["k_norm"].double()
    normed = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + EPS) * weight
    r = c["rot"]
    if r:
        i = torch.arange(r // 2, device=GPU)
        angle = s["pos"].double()[:, None] * torch.exp(-2.0 * i.double() / r * math.log(c["theta"]))
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        a, b = (i, i + r // 2) if c["pairs"] == "halves" else (2 * i, 2 * i + 1)
        z = torch.complex(normed[..., a], normed[..., b]) * turn
        normed[..., a], normed[..., b] = z.real, z.imag
    x = torch.where((heads < c["hq"] + c["hk"])[None, :, None], normed, x)
    most = s["k_out"].shape[1]
    out = {"q": x[:, : c["hq"]]}
    seq, pos = s["seq"].long(), s["pos"].long()
    for name, h in (("k", c["hq"]), ("v", c["hq"] + c["hk"])):
        full = torch.zeros(c["seqs"], most, c["hk"], c["d"], dtype=torch.float64, device=GPU)
        for b, y in enumerate(_exact_sequences(s, c, name)):
            full[b, : len(y)] = y
        full[seq, pos] = _exact_held(x[:, h: h + c["hk"]], c["cache"])
        out[name] = full
    return out


def _exact_weights(x, seen, cap, bias):
    if cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias
    x = x.masked_fill(~seen, -math.inf)
    return torch.nan_to_num(torch.softmax(x, -1), nan=0.0)  # a row that sees nothing


def _exact_attn(c, s):
    """Document by document and head by head."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    off = s["docs"].tolist()
    for a, b, p in zip(off, off[1:], s["prefix"].tolist()):
        i = torch.arange(b - a, device=GPU)
        seen = (i[None] <= i[:, None]) | (i[None] < p)
        for h in range(c["hq"]):
            kv = h // (c["hq"] // c["hk"])
            x = s["q"][a:b, h].double() @ s["k"][a:b, kv].double().T / math.sqrt(c["d"])
            bias = None if s["slopes"] is None else -s["slopes"][h].double() * (i[:, None] - i[None]).abs().double()
            out[a:b, h] = _exact_weights(x, seen, c["cap"], bias) @ s["v"][a:b, kv].double()
    return out


def _exact_decode(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    g = c["hq"] // c["hk"]
    for b, (k, v) in enumerate(zip(_exact_sequences(s, c, "k"), _exact_sequences(s, c, "v"))):
        far = torch.arange(len(k) - 1, -1, -1, device=GPU, dtype=torch.float64)
        for h in range(c["hk"]):
            heads = slice(h * g, h * g + g)
            x = s["q"][b, heads].double() @ k[:, h].T.contiguous() / math.sqrt(c["d"])
            bias = None if s["slopes"] is None else -s["slopes"][heads].double()[:, None] * far[None]
            out[b, heads] = _exact_weights(x, torch.ones_like(x, dtype=torch.bool), c["cap"], bias) @ v[:, h]
    return out


def _exact_beam(c, s):
    """The scores, group by group, from the best of each beam; the rest are choices, not computed numbers."""
    g, w = c["groups"], c["beams"]
    x = s["logits"].double().view(g, w, -1)
    out = torch.empty(g, w, dtype=torch.float64, device=GPU)
    for b in range(g):
        p = torch.log_softmax(x[b], -1)
        done = s["finished"][b] != 0
        p[done] = -math.inf
        p[done, s["eos"]] = 0.0
        out[b] = (p + s["scores"][b].double()[:, None]).flatten().topk(w).values
    return {"scores": out, "parents": None, "tokens": None, "finished": None, "table": None, "lens": None, "used": None,
            "k_spare": None, "v_spare": None}
