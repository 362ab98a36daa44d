"""What the speed of the text decoder's further operators is measured on: rotary positions of several
axes, caches that evict by accumulated attention weight, latent attention, through this library's
public entry points.

Seven kinds of pass: queries or keys rotated by (time, row, column) positions ("rotate"), the same
where a step's projections go into the paged cache ("append"); attention over packed prompts that
also adds up the weight each key got ("weigh"), and of single tokens ("single"); the eviction of
what got least from the cache ("evict"); a step of latent attention, the new tokens' latents written
and all attended to ("absorbed"); a prompt's latent attention with expanded keys and values
("expanded").

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
CODED = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def listed():
    return [
        # The next token of every beam of a page's 36 lines, four beams a line; image tokens have three axes.
        {"name": "append_beams", "kind": "append", "seqs": 144, "new": 1, "past": 300, "hq": 16, "hk": 2, "d": 128, "rot": 128,
         "axes": "24,20,20", "order": "turns", "ladder": "shared", "theta": 5e5, "pairs": "halves", "page": 16, "type": "bf16"},
        # A video's patches in an encoder: queries of 16 heads out of the packed projections, rows and columns with own frequencies.
        {"name": "rotate_video", "kind": "rotate", "n": 65521, "heads": 16, "d": 80, "first": 0, "rot": 80, "axes": "20,20",
         "order": "blocks", "ladder": "own", "theta": 1e4, "pairs": "halves", "packed": 3, "type": "bf16"},
        # A page's 36 lines packed into one row, each line's last 32 queries say what is kept.
        {"name": "weigh_lines", "kind": "weigh", "docs": 36, "most": 130, "prefix": 0.7, "hq": 16, "hk": 4, "d": 64, "cap": 0.0,
         "slopes": False, "pad": 37, "window": 32, "type": "f16"},
        # Long documents, causal but for a short prefix, every query counts.
        {"name": "weigh_long", "kind": "weigh", "docs": 2, "most": 5000, "prefix": 0.1, "hq": 32, "hk": 8, "d": 128, "cap": 0.0,
         "slopes": False, "pad": 0, "window": 0, "type": "bf16"},
        # One line's next token.
        {"name": "single_line", "kind": "single", "seqs": 1, "len": 201, "hq": 8, "hk": 8, "d": 64, "cap": 0.0, "slopes": False,
         "page": 16, "type": "f16", "cache": "f16"},
        # A batch of long documents over an 8-bit cache.
        {"name": "single_long", "kind": "single", "seqs": 16, "len": 30011, "hq": 32, "hk": 8, "d": 128, "cap": 0.0, "slopes": False,
         "page": 64, "type": "bf16", "cache": "e4m3"},
        # Lines' caches that have grown a little past what they may keep.
        {"name": "evict_lines", "kind": "evict", "seqs": 36, "len": 528, "keep": 512, "sinks": 4, "recent": 64, "hk": 4, "d": 64,
         "page": 16, "cache": "f16"},
        # Long prompts cut down to an eighth before the first token is written.
        {"name": "evict_prompts", "kind": "evict", "seqs": 8, "len": 16500, "keep": 2048, "sinks": 4, "recent": 256, "hk": 8, "d": 128,
         "page": 64, "cache": "bf16"},
        # One document's next token, a small model.
        {"name": "absorbed_one", "kind": "absorbed", "seqs": 1, "len": 900, "heads": 16, "rank": 128, "rot": 32, "page": 16, "type": "f16"},
        # A batch's next tokens, all heads of a large model on this GPU.
        {"name": "absorbed_batch", "kind": "absorbed", "seqs": 64, "len": 8191, "heads": 128, "rank": 512, "rot": 64, "page": 64,
         "type": "bf16"},
        # A page's lines in one row.
        {"name": "expanded_lines", "kind": "expanded", "docs": 36, "most": 130, "prefix": 0.7, "heads": 12, "dk": 64, "rot": 32, "dv": 64,
         "pad": 37, "type": "f16"},
        # Long documents, causal.
        {"name": "expanded_long", "kind": "expanded", "docs": 2, "most": 5000, "prefix": 0.0, "heads": 32, "dk": 128, "rot": 64, "dv": 128,
         "pad": 0, "type": "bf16"},
    ]


def draw(rng):
    """A case of the same ranges: sizes spread over their logarithm, odd ones among them, none that
    costs more than the largest listed one of its kind."""
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(max(a, b))))))

    def axes(rot):
        n, left, out = rng.choice([1, 2, 3, 3, 4]), rot // 2, []
        for k in range(n - 1):
            out.append(rng.randint(0, left // 2))
            left -= out[-1]
        return {"axes": ",".join(map(str, out + [left])), "order": rng.choice(["blocks", "turns"]), "ladder": rng.choice(["shared", "own"]),
                "theta": rng.choice([1e4, 5e5]), "pairs": rng.choice(["halves", "adjacent"])}

    kind = rng.choice(["append", "rotate", "weigh", "single", "evict", "absorbed", "expanded"])
    page, t16 = rng.choice([16, 32, 64]), rng.choice(["f16", "bf16"])
    if kind in ("append", "rotate"):
        d = rng.choice([32, 64, 64, 80, 96, 128, 128])
        rot = rng.choice([d, d, 32])
        if kind == "rotate":
            heads, packed = rng.choice([1, 2, 6, 16, 20]), rng.choice([1, 2, 3])
            return {"kind": kind, "n": log(1, min(65521, 16000000 // (heads * d))), "heads": heads, "d": d, "first": rng.choice([0, d - rot]),
                    "rot": rot, **axes(rot), "packed": packed, "type": rng.choice([t16, t16, "f32"])}
        hk = rng.choice([1, 2, 4, 8])
        c = {"kind": kind, "hk": hk, "hq": hk * rng.choice([1, 2, 4, 8]), "d": d, "rot": rot, **axes(rot), "page": page, "type": t16}
        if rng.random() < 0.4:  # a step of single tokens
            n = log(1, 200)
            c.update(seqs=n, new=1, past=log(1, min(2000, 60000 // n)))
        else:
            c.update(seqs=log(1, 8), new=log(2, 1100), past=rng.choice([0, 0, log(1, 300)]))
        return c
    if kind in ("weigh", "single"):
        hk = rng.choice([1, 2, 4, 8])
        h = {"hk": hk, "hq": hk * rng.choice([1, 2, 3, 4, 8]), "d": rng.choice([32, 64, 64, 80, 96, 128, 128])}
        if kind == "single":
            n = log(1, 200)
            return {"kind": kind, "seqs": n, "len": log(1, min(60000, 230000 // n)), **h, "cap": rng.choice([0.0, 0.0, 30.0]),
                    "slopes": rng.random() < 0.3, "page": page, "type": t16, "cache": rng.choice([t16, "i8", "e4m3"])}
        docs = log(1, 40)
        most = int(min(7000, (2.3e11 / (4 * h["hq"] * h["d"])) ** 0.5)) // docs
        return {"kind": kind, "docs": docs, "most": log(1, most), "prefix": rng.choice([0.0, 0.1, 0.5, 0.7, 1.0]), **h,
                "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.3, "pad": rng.choice([0, 0, log(1, 99)]),
                "window": rng.choice([0, 0, 1, 32, log(1, 500)]), "type": t16}
    if kind == "evict":
        n, hk, d = log(1, 150), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 96, 128])
        most = log(2, min(40000, 130000 // n))
        keep = rng.choice([max(1, most - log(1, 64)), log(1, most), max(1, most // 8)])
        sinks = min(keep, rng.choice([0, 1, 4]))
        return {"kind": kind, "seqs": n, "len": most, "keep": keep, "sinks": sinks, "recent": min(keep - sinks, rng.choice([0, 1, log(1, 500)])),
                "hk": hk, "d": d, "page": page, "cache": rng.choice(["f16", "bf16", "i8"])}
    if kind == "absorbed":
        n, heads = log(1, 150), rng.choice([1, 5, 8, 16, 16, 32, 40, 64, 128])
        return {"kind": kind, "seqs": n, "len": log(1, min(100000, 33000000 // (n * max(heads, 16)))), "heads": heads,
                "rank": rng.choice([64, 128, 256, 384, 512, 512]), "rot": rng.choice([32, 64, 64]), "page": page, "type": t16}
    docs, heads = log(1, 40), rng.choice([1, 3, 8, 12, 20, 32])
    dk, rot, dv = rng.choice([(32, 32, 32), (64, 32, 64), (64, 64, 64), (96, 32, 64), (128, 64, 128), (128, 64, 128)])
    most = int(min(7000, (2.3e11 / (2 * heads * (dk + rot + dv))) ** 0.5)) // docs
    return {"kind": kind, "docs": docs, "most": log(1, most), "prefix": rng.choice([0.0, 0.0, 0.1, 0.7, 1.0]), "heads": heads, "dk": dk,
            "rot": rot, "dv": dv, "pad": rng.choice([0, 0, log(1, 99)]), "type": t16}


# ---- sizes that follow from a case --------------------------------------------------------------
def _counts(n, most, salt):
    """n ragged lengths: the first the most, the others between a quarter of it and all of it."""
    rng = random.Random(n * 1000003 + most * 31 + salt)
    return [most] + [rng.randint(max(1, most // 4), most) for _ in range(n - 1)]


def _kv_sizes(c):
    past = _counts(c["seqs"], c["past"], 1) if c["past"] else [0] * c["seqs"]
    return past, _counts(c["seqs"], c["new"], 2)


def _evict_lens(c):
    """Half of the sequences near the most, the others anywhere up to it, as some have not grown past what they keep."""
    rng = random.Random(c["len"] * 7 + c["seqs"])
    return [c["len"]] + [rng.randint(max(1, c["len"] - c["len"] // 32) if k % 2 else 1, c["len"]) for k in range(c["seqs"] - 1)]


def _axis_pairs(c):
    return [int(v) for v in c["axes"].split(",")]


# ---- inputs --------------------------------------------------------------------------------------
def _cache(gen, c, pages):
    """A paged cache's memory, [pages][heads][page][dim] and a scale a vector for the 8-bit ones."""
    shape = (pages, c["hk"], c["page"], c["d"])
    fmt = c["cache"]
    out = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device=GPU, dtype=torch.float16)
        s = None
        if fmt == "i8":
            x = (x * 40).round().clamp(-127, 127).to(torch.int8)
        elif fmt == "e4m3":
            x = (x.float() * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            x = x.to(TYPES[fmt])
        if fmt in CODED:
            s = (0.6 + torch.rand(shape[:3], generator=gen, device=GPU)) * (0.025 if fmt == "i8" else 0.009)
        out[name], out[name + "_scale"] = x, s
    return out


def _tables(gen, lens, page):
    """Every sequence's pages, anywhere in the pool (-1 past its last), and how many pages that takes."""
    need = [-(-n // page) for n in lens]
    total, width = sum(need), max(max(need), 1)
    perm = torch.randperm(total, generator=gen, device=GPU).to(torch.int32)
    col = torch.arange(width, device=GPU)[None]
    n = torch.tensor(need, device=GPU)[:, None]
    first = torch.cumsum(n, 0) - n
    at = (first + col).clamp(max=total - 1)
    return torch.where(col < n, perm[at], -1).to(torch.int32).contiguous(), total


def _grid_positions(gen, n, axes):
    """Time, row and column of a video's patches (64 x 36 a frame), far from the start; text tokens would have all alike."""
    at = torch.arange(n, device=GPU)
    start = torch.randint(0, 20000, (axes,), generator=gen, device=GPU)
    parts = [at // 2304, at // 64 % 36, at % 64, at]
    return (torch.stack([parts[3 if axes == 1 else k] for k in range(axes)], 1) + start).to(torch.int32).contiguous()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(GPU).manual_seed(int(seed) * 7919 + 23)
    rn = lambda *shape: torch.randn(*shape, generator=gen, device=GPU)  # noqa: E731
    s = {"case": c}
    kind = c["kind"]
    i32 = dict(dtype=torch.int32, device=GPU)
    t = TYPES[c["type"]] if "type" in c else None
    if kind == "append":
        past, new = _kv_sizes(c)
        s["table"], pages = _tables(gen, [p + n for p, n in zip(past, new)], c["page"])
        s["cache"] = _cache(gen, {**c, "cache": c["type"]}, pages)
        n, width = sum(new), (c["hq"] + 2 * c["hk"]) * c["d"]
        s["qkv"] = (rn(n, width) * (0.3 + rn(1, width).abs())).to(t)  # channels of unlike size
        s["seq"] = torch.repeat_interleave(torch.arange(len(new), device=GPU), torch.tensor(new, device=GPU)).to(torch.int32)
        s["pos"] = torch.cat([torch.arange(p, p + k, **i32) for p, k in zip(past, new)])
        s["at"] = _grid_positions(gen, n, len(_axis_pairs(c)))
        s["q_norm"], s["k_norm"] = 1 + 0.2 * rn(c["d"]), 1 + 0.2 * rn(c["d"])
        s["q"] = torch.empty(n, c["hq"], c["d"], dtype=t, device=GPU)
        s["k"] = torch.empty(n, c["hk"], c["d"], dtype=t, device=GPU)
    elif kind == "rotate":
        n = c["n"]
        s["wide"] = rn(n, c["packed"], c["heads"], c["d"]).to(t)  # the projections of queries, keys and values as they come
        s["x"] = s["wide"][:, 0]
        s["at"] = _grid_positions(gen, n, len(_axis_pairs(c)))
        s["out"] = torch.empty(n, c["heads"], c["d"], dtype=t, device=GPU)
    elif kind in ("weigh", "expanded"):
        lens = _counts(c["docs"], c["most"], 3)
        n = sum(lens) + c["pad"]
        off = [0]
        for k in lens:
            off.append(off[-1] + k)
        s["docs"] = torch.tensor(off, **i32)
        s["prefix"] = torch.tensor([int(k * c["prefix"]) for k in lens], **i32)
        if kind == "weigh":
            s["q"], s["k"], s["v"] = ((rn(n, h, c["d"]) * a).to(t) for h, a in ((c["hq"], 1.5), (c["hk"], 1.0), (c["hk"], 1.0)))
            s["slopes"] = _slopes(c)
            s["out"] = torch.empty_like(s["q"])
            s["weights"] = torch.rand(c["docs"], c["hk"], c["most"], generator=gen, device=GPU)
        else:
            s["q"] = (rn(n, c["heads"], c["dk"] + c["rot"]) * 1.3).to(t)
            up = rn(n, c["heads"], c["dk"] + c["dv"]).to(t)  # one product expands keys and values
            s["k"], s["v"] = up[..., : c["dk"]], up[..., c["dk"]:]
            s["r"] = rn(n, 512 + c["rot"]).to(t)[:, 512:]  # beside the latents
            s["out"] = torch.empty(n, c["heads"], c["dv"], dtype=t, device=GPU)
    elif kind == "single":
        lens = _counts(c["seqs"], c["len"], 4)
        s["table"], pages = _tables(gen, lens, c["page"])
        s["cache"] = _cache(gen, c, pages)
        s["lens"] = torch.tensor(lens, **i32)
        s["q"] = (rn(c["seqs"], c["hq"], c["d"]) * 1.5).to(t)
        s["slopes"] = _slopes(c)
        s["out"] = torch.empty_like(s["q"])
        s["weights"] = torch.rand(c["seqs"], c["hk"], c["len"], generator=gen, device=GPU)
    elif kind == "evict":
        lens = _evict_lens(c)
        s["table"], pages = _tables(gen, lens, c["page"])
        s["cache"] = _cache(gen, c, pages)
        s["lens"] = torch.tensor(lens, **i32)
        shape = (c["seqs"], c["hk"], c["len"])
        # A few keys have most of the weight; whole tokens of none among the last.
        s["weights"] = torch.rand(shape, generator=gen, device=GPU) ** 6 * (torch.rand(shape, generator=gen, device=GPU) > 0.1)
        # What an earlier eviction left holds tokens of anywhere before the newest, the places after it are new.
        seen = (s["lens"].float() * torch.rand(c["seqs"], generator=gen, device=GPU)).int()
        p = torch.arange(c["len"], **i32)
        s["newest"] = s["lens"] + 700
        s["held"] = torch.where(p < seen[:, None, None], p + (torch.rand(shape, generator=gen, device=GPU) * 100).int(), -1).contiguous()
        s["weights_out"], s["held_out"] = torch.empty_like(s["weights"]), torch.empty_like(s["held"])
        s["lens_out"] = torch.empty_like(s["lens"])
    else:
        lens = _counts(c["seqs"], c["len"], 6)
        s["table"], pages = _tables(gen, lens, c["page"])
        width = c["rank"] + c["rot"]
        s["pool"] = rn(pages, c["page"], width).to(t)
        s["lens"] = torch.tensor(lens, **i32)
        s["x"] = (rn(c["seqs"], width) * (0.3 + rn(1, width).abs())).to(t)
        s["norm"] = 1 + 0.2 * rn(c["rank"])
        s["seq"], s["pos"] = torch.arange(c["seqs"], **i32), s["lens"] - 1
        s["q"] = rn(c["seqs"], c["heads"], width).to(t)
        s["out"] = torch.empty(c["seqs"], c["heads"], c["rank"], dtype=t, device=GPU)
    return s


def _slopes(c):
    """Distance slopes in a geometric row, one a head."""
    if not c["slopes"]:
        return None
    return 2.0 ** (-8.0 * (1 + torch.arange(c["hq"], device=GPU, dtype=torch.float32)) / c["hq"])


def _latent_scale(c):
    return (c["rank"] / 4 + c["rot"]) ** -0.5 if "rank" in c else (c["dk"] + c["rot"]) ** -0.5


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "rotate": _plain_rotate, "weigh": _plain_weigh, "single": _plain_single, "evict": _plain_evict,
            "absorbed": _plain_absorbed, "expanded": _plain_expanded}[s["case"]["kind"]](s)


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
        c = s["case"]
        if c["kind"] == "absorbed":
            s["handle"] = ocrhip.LatentCache(ctx, s["pool"].shape[0], c["page"], c["rank"], c["rot"], c["type"], memory=s["pool"])
        else:
            m = s["cache"]
            pages, heads, page, dim = m["k"].shape
            s["handle"] = ocrhip.KvCache(ctx, pages, page, heads, dim, c.get("cache", c.get("type")),
                                         memory=(m["k"], m["v"], m["k_scale"], m["v_scale"]))
    return s["handle"]


def _turns(s):
    """How a program names its axes."""
    if "turns" not in s:
        c = s["case"]
        s["turns"] = {"rot": c["rot"], "theta": c["theta"], "pairs": c["pairs"], "axes": tuple(_axis_pairs(c)), "order": c["order"],
                      "ladder": c["ladder"]}
    return s["turns"]


def _run_own(s):
    ocrhip, ctx = _library()
    c = s["case"]
    kind = c["kind"]
    if kind == "append":
        _handle(s).append(s["table"], s["seq"], s["pos"], s["qkv"], s["q"], s["k"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                          at=s["at"], **_turns(s))
        return {"q": s["q"], "k": s["k"], "k_pool": s["cache"]["k"], "v_pool": s["cache"]["v"]}
    if kind == "rotate":
        ocrhip.rotate(ctx, s["x"], s["at"], s["out"], first=c["first"], **_turns(s))
        return s["out"]
    if kind == "weigh":
        ocrhip.attention(ctx, s["q"], s["k"], s["v"], s["out"], s["docs"], prefix=s["prefix"], scale=c["d"] ** -0.5, cap=c["cap"],
                         slopes=s["slopes"], weights=s["weights"], window=c["window"] or None)
        return {"out": s["out"], "weights": s["weights"]}
    if kind == "single":
        _handle(s).attend(s["table"], s["lens"], s["q"], s["out"], scale=c["d"] ** -0.5, cap=c["cap"], slopes=s["slopes"],
                          weights=s["weights"])
        return {"out": s["out"], "weights": s["weights"]}
    if kind == "evict":
        _handle(s).evict(s["table"], s["lens"], s["newest"], s["weights"], s["held"], c["keep"], s["lens_out"], first=c["sinks"],
                         recent=c["recent"], weights_out=s["weights_out"], held_out=s["held_out"])
        return _evict_outputs(s, s["lens_out"], s["weights_out"], s["held_out"])
    if kind == "absorbed":
        _handle(s).append(s["table"], s["seq"], s["pos"], s["x"], norm=s["norm"], eps=EPS)
        _handle(s).attend(s["table"], s["lens"], s["q"], s["out"], scale=_latent_scale(c))
        return {"out": s["out"], "pool": s["pool"]}
    ocrhip.latent_attention(ctx, s["q"], s["k"], s["r"], s["v"], s["out"], s["docs"], prefix=s["prefix"], scale=_latent_scale(c))
    return s["out"]


def _evict_outputs(s, lens, weights, held):
    m = s["cache"]
    out = {"lens": lens, "weights": weights, "held": held, "k": m["k"], "v": m["v"]}
    if m["k_scale"] is not None:
        out.update(k_scale=m["k_scale"], v_scale=m["v_scale"])
    return out


# ---- the plain forms -----------------------------------------------------------------------------
def _frequencies(c):
    """Every pair's axis and frequency (float64)."""
    sizes = _axis_pairs(c)
    axis, index = [], []
    if c["order"] == "blocks":
        axis = [a for a, n in enumerate(sizes) for _ in range(n)]
        index = [j for n in sizes for j in range(n)]
    else:  # one of each axis in turn, as long as it has pairs left
        both = sorted((j, a) for a, n in enumerate(sizes) for j in range(n))
        axis, index = [a for _, a in both], [j for j, _ in both]
    half = c["rot"] // 2
    share = [(p / half) if c["ladder"] == "shared" else j / sizes[a] for p, (a, j) in enumerate(zip(axis, index))]
    return torch.tensor(axis, device=GPU), c["theta"] ** -torch.tensor(share, dtype=torch.float64, device=GPU)


def _turned(x, at, c):
    """x [n][heads][rot] float32 rotated by the positions at [n][axes]; the angles in float64."""
    axis, freq = _frequencies(c)
    angle = (at.double()[:, axis] * freq)[:, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    y, h = torch.empty_like(x), c["rot"] // 2
    if c["pairs"] == "halves":
        a, b = x[..., :h], x[..., h:]
        y[..., :h], y[..., h:] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y[..., 0::2], y[..., 1::2] = a * cos - b * sin, b * cos + a * sin
    return y


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_rotate(s):
    c = s["case"]
    f, r = c["first"], c["rot"]
    y = s["x"].float()
    y[..., f: f + r] = _turned(y[..., f: f + r].clone(), s["at"], c)
    return y.to(TYPES[c["type"]])


def _plain_append(s):
    c, m, t = s["case"], s["cache"], TYPES[s["case"]["type"]]
    n, hq, hk, d, r = s["qkv"].shape[0], c["hq"], c["hk"], c["d"], c["rot"]
    q, k, v = s["qkv"].float().view(n, hq + 2 * hk, d).split([hq, hk, hk], 1)
    q, k = _norm(q, s["q_norm"]), _norm(k, s["k_norm"])
    q = torch.cat([_turned(q[..., :r], s["at"], c), q[..., r:]], -1).to(t)
    k = torch.cat([_turned(k[..., :r], s["at"], c), k[..., r:]], -1).to(t)
    pos = s["pos"].long()
    page, row = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    m["k"][page, :, row], m["v"][page, :, row] = k, v.to(t)
    return {"q": q, "k": k, "k_pool": m["k"], "v_pool": m["v"]}


def _softmax_rows(x, seen):
    """exp(x - max) over its sum, along the last axis, nothing where not seen; rows that see nothing weigh nothing."""
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1)


def _cap(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _document_masks(s, c):
    """Which tokens see which [n][n], every token's document (the last for those outside) and whether it has one."""
    at = torch.arange(s["q"].shape[0], device=GPU)
    doc = torch.searchsorted(s["docs"], at.int(), right=True) - 1
    inside, doc = doc < c["docs"], doc.clamp(max=c["docs"] - 1)
    seen = (doc[:, None] == doc[None]) & inside[:, None] & inside[None]
    seen &= (at[None] <= at[:, None]) | (at[None] < (s["docs"][:-1] + s["prefix"])[doc][:, None])
    return seen, doc, inside


def _plain_weigh(s):
    c = s["case"]
    n, hk, d, g = s["q"].shape[0], c["hk"], c["d"], c["hq"] // c["hk"]
    q = s["q"].float().view(n, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * n, d)
    k, v = (s[x].float().transpose(0, 1).contiguous() for x in ("k", "v"))
    x = _cap(torch.matmul(q, k.transpose(1, 2).contiguous()).view(hk, g, n, n) * d ** -0.5, c["cap"])
    at = torch.arange(n, device=GPU)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(hk, g, 1, 1) * (at[:, None] - at[None]).abs()
    seen, doc, inside = _document_masks(s, c)
    p = _softmax_rows(x, seen)
    del x
    o = torch.matmul(p.view(hk, g * n, n), v).view(hk, g, n, d).permute(2, 0, 1, 3).reshape(n, c["hq"], d).to(TYPES[c["type"]])
    counts = at >= s["docs"][1:][doc] - (c["window"] or n)  # the queries whose weights are added up
    # A key's share of all queries' attention, the group's heads together.
    got = torch.matmul((counts & inside).float()[None, None], p.sum(1))[:, 0]
    row, place = doc[inside], (at - s["docs"][:-1][doc])[inside]
    s["weights"][row, :, place] += got[:, inside].T
    return {"out": o, "weights": s["weights"]}


def _values(cache, name, fmt, table):
    """The vectors of every sequence's pages, float32 [sequences][positions][heads][d]."""
    x = cache[name][table.clamp(min=0).long()]
    x = (x.view(torch.float8_e4m3fn) if fmt == "e4m3" else x).float()
    if fmt in CODED:
        x = x * cache[name + "_scale"][table.clamp(min=0).long()][..., None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_single(s):
    c, m = s["case"], s["cache"]
    n, hk, d, g = c["seqs"], c["hk"], c["d"], c["hq"] // c["hk"]
    k, v = (_values(m, x, c["cache"], s["table"]).transpose(1, 2).contiguous() for x in ("k", "v"))
    q = s["q"].float().view(n, hk, g, d)
    x = _cap(torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5, c["cap"])
    at = torch.arange(k.shape[2], device=GPU)[None, None, None]
    last = s["lens"].view(n, 1, 1, 1) - 1
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hk, g, 1) * (last - at)
    p = _softmax_rows(x, at <= last)
    s["weights"] += p.sum(2)[:, :, : c["len"]]
    return {"out": torch.matmul(p, v).reshape(n, c["hq"], d).to(TYPES[c["type"]]), "weights": s["weights"]}


def _plain_evict(s):
    c, m, page = s["case"], s["cache"], s["case"]["page"]
    most, i = c["len"], torch.int32
    p = torch.arange(most, device=GPU)
    n = s["lens"].long()[:, None, None]
    lens = s["lens"].clamp(max=c["keep"])
    left = lens.long()[:, None, None]
    newest = s["newest"].long()[:, None, None]
    held = torch.where(s["held"] >= 0, s["held"].long(), newest - (n - 1 - p))
    safe = (held < c["sinks"]) | (held > newest - c["recent"])
    key = torch.where(safe, math.inf, s["weights"].double())
    key = torch.where(p < n, key, -math.inf)
    order = torch.sort(key, dim=2, descending=True, stable=True).indices
    kept = torch.zeros_like(key, dtype=torch.bool).scatter_(2, order, (p < left).expand_as(key))
    holes = torch.where(~kept & (p < left), p, most).sort(2).values
    moved = torch.where(kept & (p >= left), p, most).sort(2).values
    source = torch.arange(most + 1, device=GPU).expand(c["seqs"], c["hk"], -1).clone().scatter_(2, holes, moved)[..., :most]
    weights = torch.where(p < left, s["weights"].gather(2, source), 0)
    held = torch.where(p < left, held.gather(2, source), -1).to(i)
    # The vectors of the moved places, to the holes.
    row, head, to = torch.nonzero((source != p) & (p < left), as_tuple=True)
    at = source[row, head, to]
    src, dst = s["table"][row, at // page].long(), s["table"][row, to // page].long()
    for name in ("k", "v", "k_scale", "v_scale"):
        if m[name] is not None:
            m[name][dst, head, to % page] = m[name][src, head, at % page]
    return _evict_outputs(s, lens, weights, held)


def _plain_absorbed(s):
    c, rank = s["case"], s["case"]["rank"]
    x = s["x"].float()
    turn = {"rot": c["rot"], "axes": str(c["rot"] // 2), "order": "blocks", "ladder": "shared", "theta": 1e4, "pairs": "halves"}
    new = torch.cat([_norm(x[:, :rank], s["norm"]), _turned(x[:, None, rank:], s["pos"][:, None], turn)[:, 0]], 1).to(TYPES[c["type"]])
    pos = s["pos"].long()
    s["pool"][s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]] = new
    kv = s["pool"][s["table"].clamp(min=0).long()].flatten(1, 2).float()
    sc = torch.matmul(s["q"].float(), kv.transpose(1, 2).contiguous()) * _latent_scale(c)
    p = _softmax_rows(sc, torch.arange(kv.shape[1], device=GPU)[None, None] < s["lens"].view(-1, 1, 1))
    return {"out": torch.matmul(p, kv[..., :rank].contiguous()).to(TYPES[c["type"]]), "pool": s["pool"]}


def _plain_expanded(s):
    c = s["case"]
    n, h, dk = s["q"].shape[0], c["heads"], c["dk"]
    q = s["q"].float().transpose(0, 1).contiguous()
    k = torch.cat([s["k"].float(), s["r"].float()[:, None].expand(n, h, c["rot"])], 2).permute(1, 2, 0).contiguous()
    x = torch.matmul(q, k) * _latent_scale(c)
    p = _softmax_rows(x, _document_masks(s, c)[0])
    del x
    return torch.matmul(p, s["v"].float().transpose(0, 1).contiguous()).transpose(0, 1).contiguous().to(TYPES[c["type"]])


# ---- the work ------------------------------------------------------------------------------------
def _pairs_seen(lens, prefix):
    total = 0
    for k in lens:
        p = int(k * prefix)
        total += p * p + (k * (k + 1) - p * (p + 1)) // 2  # prefix rows see the prefix, the others their past
    return total


def work(case):
    c, kind = case, case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]] if "type" in c else 2
    if kind == "append":
        n = sum(_kv_sizes(c)[1])
        width = (c["hq"] + 2 * c["hk"]) * c["d"]
        # The projections in; queries, keys and the cache's keys and values out.
        return {"bytes": n * (width + (c["hq"] + 3 * c["hk"]) * c["d"]) * size + 4 * n * (2 + len(_axis_pairs(c))), "flops": 10 * n * width}
    if kind == "rotate":
        values = c["n"] * c["heads"] * c["d"]
        return {"bytes": 2 * values * size + 4 * c["n"] * len(_axis_pairs(c)), "flops": 6 * values}
    if kind in ("weigh", "expanded"):
        lens = _counts(c["docs"], c["most"], 3)
        n, pairs = sum(lens) + c["pad"], _pairs_seen(lens, c["prefix"])
        if kind == "expanded":
            row = c["heads"] * (c["dk"] + c["rot"] + c["dk"] + 2 * c["dv"]) + c["rot"]
            return {"bytes": n * row * size, "flops": 2 * pairs * c["heads"] * (c["dk"] + c["rot"] + c["dv"])}
        # The scores a second time, once their sums are known, for the queries that count.
        again = 0
        for k in lens:
            p, w = int(k * c["prefix"]), min(c["window"] or k, k)
            first = k - w
            for_prefix = max(0, p - first)
            again += for_prefix * p + sum(range(max(first, p) + 1, k + 1))
        return {"bytes": n * 2 * (c["hq"] + c["hk"]) * c["d"] * size + 8 * sum(lens) * c["hk"],
                "flops": (4 * pairs + 2 * again) * c["hq"] * c["d"]}
    if kind == "single":
        total = sum(_counts(c["seqs"], c["len"], 4))
        held = c["d"] * (1 if c["cache"] in CODED else 2) + (4 if c["cache"] in CODED else 0)
        return {"bytes": total * c["hk"] * (2 * held + 8) + 2 * c["seqs"] * c["hq"] * c["d"] * size, "flops": 4 * total * c["hq"] * c["d"]}
    if kind == "evict":
        lens = _evict_lens(c)
        held = c["d"] * (1 if c["cache"] in CODED else 2) + (4 if c["cache"] in CODED else 0)
        # Weights and positions in and out. How many vectors move depends on the values: as many as at random.
        moved = sum((n - c["keep"]) * c["keep"] / n for n in lens if n > c["keep"])
        return {"bytes": c["hk"] * (sum(lens) * 8 + c["seqs"] * c["len"] * 8 + moved * 4 * held), "flops": 4 * c["hk"] * sum(lens)}
    total = sum(_counts(c["seqs"], c["len"], 6))
    width = c["rank"] + c["rot"]
    return {"bytes": total * width * size + c["seqs"] * (c["heads"] * (width + c["rank"]) + 2 * width) * size,
            "flops": 2 * total * c["heads"] * (width + c["rank"])}


# ---- the definitions in float64 ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "rotate": _exact_rotate, "weigh": _exact_weigh, "single": _exact_single, "evict": _exact_evict,
            "absorbed": _exact_absorbed, "expanded": _exact_expanded}[case["kind"]](case, s)


def _exact_turn(x, at, c):
    """x [n][heads][rot] float64, pair by pair as complex numbers."""
    sizes, half = _axis_pairs(c), c["rot"] // 2
    used, axis, y = [0] * len(sizes), 0, x.clone()
    for p in range(half):
        if c["order"] == "blocks":
            while used[axis] == sizes[axis]:
                axis += 1
            a = axis
        else:  # the axis that has given fewest so far and has some left
            a = min((k for k in range(len(sizes)) if used[k] < sizes[k]), key=lambda k: (used[k], k))
        power = p / half if c["ladder"] == "shared" else used[a] / sizes[a]
        used[a] += 1
        angle = at[:, a].double() * math.exp(-power * math.log(c["theta"]))
        i, j = (p, p + half) if c["pairs"] == "halves" else (2 * p, 2 * p + 1)
        z = torch.complex(x[..., i], x[..., j]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., i], y[..., j] = z.real, z.imag
    return y


def _exact_rotate(c, s):
    y = s["x"].double()
    f, r = c["first"], c["rot"]
    y[..., f: f + r] = _exact_turn(y[..., f: f + r].clone(), s["at"], c)
    return y


def _exact_normed(x, w):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()


def _exact_append(c, s):
    x = s["qkv"].double().reshape(-1, c["hq"] + 2 * c["hk"], c["d"])
    hq, hk, r = c["hq"], c["hk"], c["rot"]
    q, k, v = _exact_normed(x[:, :hq], s["q_norm"]), _exact_normed(x[:, hq: hq + hk], s["k_norm"]), x[:, hq + hk:]
    for y in (q, k):
        y[..., :r] = _exact_turn(y[..., :r].clone(), s["at"], c)
    pools = []
    for name, y in (("k", k), ("v", v)):
        pool = s["cache"][name].double()
        where = s["pos"].long()
        pages = torch.gather(s["table"][s["seq"].long()], 1, (where // c["page"])[:, None])[:, 0].long()
        pool.transpose(1, 2)[pages, where % c["page"]] = y
        pools.append(pool)
    return {"q": q, "k": k, "k_pool": pools[0], "v_pool": pools[1]}


def _exact_softmax(x, seen, cap, bias):
    if cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias
    return torch.nan_to_num(torch.softmax(x.masked_fill(~seen, -math.inf), -1), nan=0.0)  # a row that sees nothing


def _exact_documents(c, s):
    off = s["docs"].tolist()
    for d, (a, b, p) in enumerate(zip(off, off[1:], s["prefix"].tolist())):
        i = torch.arange(b - a, device=GPU)
        yield d, a, b, i, (i[None] <= i[:, None]) | (i[None] < p)


def _exact_weigh(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    weights = s["weights"].double()
    g = c["hq"] // c["hk"]
    for d, a, b, i, seen in _exact_documents(c, s):
        for h in range(c["hq"]):
            x = s["q"][a:b, h].double() @ s["k"][a:b, h // g].double().T / math.sqrt(c["d"])
            bias = None if s["slopes"] is None else -s["slopes"][h].double() * (i[:, None] - i[None]).abs().double()
            p = _exact_softmax(x, seen, c["cap"], bias)
            out[a:b, h] = p @ s["v"][a:b, h // g].double()
            weights[d, h // g, : b - a] += p[-min(c["window"] or b - a, b - a):].sum(0)
    return {"out": out, "weights": weights}


def _exact_sequence(s, c, name, row, n):
    """A sequence's float64 [positions][heads][d], from the pages as they are."""
    pages = s["table"][row, : -(-n // c["page"])].long()
    x = s["cache"][name][pages]
    x = (x.view(torch.float8_e4m3fn).float() if c["cache"] == "e4m3" else x).double()
    if c["cache"] in CODED:
        x = x * s["cache"][name + "_scale"][pages].double().unsqueeze(-1)
    return x.transpose(1, 2).flatten(0, 1)[:n]


def _exact_single(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    weights = s["weights"].double()
    g = c["hq"] // c["hk"]
    for b, n in enumerate(s["lens"].tolist()):
        k, v = (_exact_sequence(s, c, x, b, n) for x in ("k", "v"))
        far = torch.arange(n - 1, -1, -1, device=GPU, dtype=torch.float64)
        for h in range(c["hk"]):
            heads = slice(h * g, h * g + g)
            x = s["q"][b, heads].double() @ k[:, h].T.contiguous() / math.sqrt(c["d"])
            bias = None if s["slopes"] is None else -s["slopes"][heads].double()[:, None] * far[None]
            p = _exact_softmax(x, torch.ones_like(x, dtype=torch.bool), c["cap"], bias)
            out[b, heads] = p @ v[:, h]
            weights[b, h, :n] += p.sum(0)
    return {"out": out, "weights": weights}


def _exact_evict(c, s):
    """Sequence by sequence and head by head; what is copied is as exact as it was."""
    coded = c["cache"] in CODED
    floats = {k: v.double() for k, v in s["cache"].items() if v is not None and (k.endswith("scale") or not coded)}
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device=GPU)
    for b, (n, newest) in enumerate(zip(s["lens"].tolist(), s["newest"].tolist())):
        left = min(n, c["keep"])
        row = s["table"][b].long()
        for h in range(c["hk"]):
            w = s["weights"][b, h, :n].double()
            held = s["held"][b, h, :n].long()
            new = held < 0
            held[new] = (torch.arange(n, device=GPU) + newest - n + 1)[new]
            w2 = w.clone()
            w2[(held < c["sinks"]) | (held > newest - c["recent"])] = math.inf
            best = torch.sort(w2, descending=True, stable=True).indices[:left]
            stay = torch.zeros(n, dtype=torch.bool, device=GPU)
            stay[best] = True
            to = torch.nonzero(~stay[:left])[:, 0]
            at = left + torch.nonzero(stay[left:])[:, 0]
            w[to] = w[at]
            weights[b, h, :left] = w[:left]
            for name, y in floats.items():
                y[row[to // c["page"]], h, to % c["page"]] = y[row[at // c["page"]], h, at % c["page"]]
    out = {"lens": None, "weights": weights, "held": None, "k": floats.get("k"), "v": floats.get("v")}
    if coded:
        out.update(k_scale=floats["k_scale"], v_scale=floats["v_scale"])
    return out


def _exact_absorbed(c, s):
    rank, pool = c["rank"], s["pool"].double()
    x = s["x"].double()
    turn = {"rot": c["rot"], "axes": str(c["rot"] // 2), "order": "blocks", "ladder": "shared", "theta": 1e4, "pairs": "halves"}
    x = torch.cat([_exact_normed(x[:, :rank], s["norm"]), _exact_turn(x[:, None, rank:], s["pos"][:, None], turn)[:, 0]], 1)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=GPU)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : -(-n // c["page"])].long()
        kv = pool[pages].flatten(0, 1)[:n]
        kv[n - 1] = x[b].to(s["pool"].dtype).double()  # attention reads what the cache holds
        pool[pages[-1], (n - 1) % c["page"]] = x[b]
        out[b] = torch.softmax(s["q"][b].double() @ kv.T.contiguous() * _latent_scale(c), -1) @ kv[:, :rank].contiguous()
    return {"out": out, "pool": pool}


def _exact_expanded(c, s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=GPU)
    dk = c["dk"]
    for _, a, b, _, seen in _exact_documents(c, s):
        for h in range(c["heads"]):
            q = s["q"][a:b, h].double()
            x = q[:, :dk] @ s["k"][a:b, h].double().T.contiguous() + q[:, dk:] @ s["r"][a:b].double().T.contiguous()
            out[a:b, h] = _exact_softmax(x * _latent_scale(c), seen, 0.0, None) @ s["v"][a:b, h].double()
    return out
