"""The text decoder's operators over the whole range of what they take: caps far over the scores,
queries and value scales of very different size beside each other, scales and codes to the last
bit. Against float64 (oracle/text.py). Tolerances count roundings: half a step of a type is EPS / 2
of the value; weights are rounded once to 16 bits, an error of the sum of p |v|, an 8-bit cache's scaled ones once more,
the output once. Scores are float32: 2^-20 of the largest that weighs anything, which the exponential passes on to the weights."""
import numpy as np
import pytest
import torch

import ocrhip
from oracle import text as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rn(g, *shape):
    return torch.randn(*shape, generator=g)


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to("cuda")


def host(x):
    torch.cuda.synchronize()
    return x.cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()


def close(got, want, size, top, eps, roundings=2):
    tol = (roundings * eps / 2 + 2.0 ** -18 + 2.0 ** -20 * top) * size + eps / 2 * np.abs(want) * (1 + eps) + 2.0 ** -24
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


def prompt(ctx, q, k, v, **kw):
    out = torch.full_like(q, 9.0)
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, **kw)
    ctx.synchronize()
    return host(out)


def single(ctx, cache, table, lens, q, **kw):
    out = torch.full_like(q, 9.0)
    t, n = i32(table), i32(lens)
    torch.cuda.synchronize()
    cache.attend(t, n, q, out, **kw)
    ctx.synchronize()
    return host(out)


def held(ctx, fmt, k, v, ks=None, vs=None, page=16):
    """(cache, table, k, v): one sequence whose vectors k, v [n][heads][dim] are codes (8-bit types, with
    scales [n][heads]) or values; the float64 values they stand for."""
    n, heads, dim = k.shape
    pages = -(-n // page)
    mem, val = [], []
    for x, s in ((k, ks), (v, vs)):
        if fmt == "i8":
            x = x.to(torch.int8)
            f = x.double()
        elif fmt == "e4m3":
            x = x.float().to(torch.float8_e4m3fn)
            f = x.float().double()
            x = x.view(torch.uint8)
        else:
            x = x.to(TYPES[fmt])
            f = x.double()
        m = torch.zeros(pages * page, heads, dim, dtype=x.dtype)
        m[:n] = x
        mem.append(m.view(pages, page, heads, dim).transpose(1, 2).contiguous().cuda())
        if fmt in plain.QMAX:
            m = torch.zeros(pages * page, heads)
            m[:n] = s
            mem.append(m.view(pages, page, heads).transpose(1, 2).contiguous().cuda())
            f = f * s.double()[..., None]
        else:
            mem.append(None)
        val.append(f.numpy())
    cache = ocrhip.KvCache(ctx, pages, page, heads, dim, fmt, memory=(mem[0], mem[2], mem[1], mem[3]))
    return cache, [list(range(pages))], val[0], val[1]


CAPS = [(-0.3, 0.0), (0.0, 0.0), (1e-30, 0.0), (-0.2, 4.0), (2.0, 30.0), (0.05, 1000.0), (0.1, 1e-3), (1e3, 1e-2), (0.1, 1e4), (0.1, 1e6),
        (0.1, 1e8), (0.1, 1e20), (0.1, 3e38), (0.1, float(np.finfo(np.float32).max)), (0.1, 1e-40)]


@pytest.mark.parametrize("fmt,ty", [("f16", "f16"), ("bf16", "bf16"), ("i8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("dim", [128, 15])
@pytest.mark.parametrize("scale,cap", CAPS)
def test_single_tokens_of_any_cap(ctx, fmt, ty, dim, scale, cap):
    """Scores of a few units under caps from nothing to the largest float, by the tiles (128) and by the formula (15)."""
    g = gen(41)
    n = 300
    k, v = ((rn(g, n, 2, dim) * (40 if fmt == "i8" else 1)).round() if fmt in plain.QMAX else rn(g, n, 2, dim) for _ in range(2))
    s = [0.02 * (0.5 + torch.rand(n, 2, generator=g)) for _ in range(2)] if fmt in plain.QMAX else [None, None]
    cache, table, kf, vf = held(ctx, fmt, k, v, *s)
    q = rn(g, 1, 4, dim).to(TYPES[ty]).cuda()
    got = single(ctx, cache, table, [n], q, scale=scale, cap=cap)
    want, size, top = plain.attention(host(q), kf, vf, ([0], [n]), scale, cap, pos=[n - 1])
    close(got, want, size, min(top, cap) if cap else top, EPS[ty], 3)


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("scale,cap", CAPS[8:])
def test_prompts_of_any_cap(ctx, ty, scale, cap):
    g = gen(42)
    q, k, v = (rn(g, 200, h, 128).to(TYPES[ty]).cuda() for h in (4, 2, 2))
    got = prompt(ctx, q, k, v, scale=scale, cap=cap)
    want, size, top = plain.attention(host(q), host(k), host(v), plain.key_ranges(200, None, None), scale, cap)
    close(got, want, size, min(top, cap), EPS[ty])


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [1e4, 1e6])
@pytest.mark.parametrize("form", ["prompt", "single"])
@pytest.mark.parametrize("bias", [False, True])
def test_capped_scores_of_very_different_size(ctx, ty, cap, form, bias):
    """Scores of a few units beside some far under them, past a third of the cap, in every tile: those
    weigh nothing, and the others must not feel the cap."""
    g = gen(43)
    n, dim = 260, 64
    q, k = torch.zeros(n, 2, dim), torch.zeros(n, 1, dim)
    q[..., 0] = 1.0
    k[..., 0] = (torch.rand(n, 1, generator=g) * 4).to(TYPES[ty]).float()
    k[5::9, :, 0] = -2.0 ** 15
    v = rn(g, n, 1, dim)
    q, k, v = (x.to(TYPES[ty]) for x in (q, k, v))
    scale = cap / 2.0 ** 16  # half the cap
    k = torch.where(k > -1000, (k.float() / scale).to(TYPES[ty]), k)  # the others: up to four units
    sl = torch.tensor([0.02, 0.01]) if bias else None
    kw = dict(scale=scale, cap=cap, slopes=None if sl is None else sl.cuda())
    rows = [0, 4, 60, 199, 259]
    want, size, _ = plain.attention(q.double().numpy()[rows], k.double().numpy(), v.double().numpy(), ([0] * 5, [r + 1 for r in rows]), scale, cap,
                                    None if sl is None else sl.numpy(), pos=rows)
    if form == "prompt":
        got = prompt(ctx, q.cuda(), k.cuda(), v.cuda(), **kw)[rows]
    else:
        cache, table, *_ = held(ctx, ty, k, v)
        got = np.concatenate([single(ctx, cache, table, [r + 1], q[r:r + 1].cuda(), **kw) for r in rows])
    close(got, want, size, 4.0, EPS[ty], 3)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("hq", [4, 16, 24])
def test_queries_of_very_different_size(ctx, fmt, hq):
    """bfloat16 heads of every size over one key head, each with scores of order one: a head's rounding is
    its own, and an infinite one's is nobody else's."""
    g = gen(44)
    n, dim = 300, 64
    k, v = ((rn(g, n, 1, dim) * 40).round() for _ in range(2))
    s = [0.02 * (0.5 + torch.rand(n, 1, generator=g)) for _ in range(2)]
    cache, table, kf, vf = held(ctx, fmt, k, v, *s)
    q = rn(g, 1, hq, dim)
    q[:, 0] *= 2.0 ** 20
    q[:, 2] *= 2.0 ** 10
    q = q.bfloat16()
    def check(got, heads):
        for h in heads:
            want, size, top = plain.attention(q.double().numpy()[:, h:h + 1], kf, vf, ([0], [n]), dim ** -0.5, pos=[n - 1])
            close(got[:, h:h + 1], want, size, top, EPS["bf16"], 3)

    check(single(ctx, cache, table, [n], q.cuda()), range(1, hq))
    q[:, 0, 3] = float("inf")
    q[:, 1, 5] = float("nan")
    got = single(ctx, cache, table, [n], q.cuda())
    assert np.isnan(got[:, 1]).all()
    check(got, range(2, hq))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("up", [-126, -100, 100, 116, 120, 126])
def test_queries_near_the_ends_of_bfloat16(ctx, fmt, up):
    g = gen(45)
    n, dim = 100, 64
    k, v = ((rn(g, n, 1, dim) * 40).round() for _ in range(2))
    # Scores of order one: 2^up of the queries, 2^-(up / 2) each of the keys' scales and the scores' own.
    ks = 0.02 * 2.0 ** (-up / 2) * (0.5 + torch.rand(n, 1, generator=g))
    vs = 0.02 * (0.5 + torch.rand(n, 1, generator=g))
    cache, table, kf, vf = held(ctx, fmt, k, v, ks, vs)
    q = (rn(g, 1, 4, dim).clamp(-1.9, 1.9).double() * 2.0 ** up).bfloat16()
    scale = dim ** -0.5 * 2.0 ** (-up / 2)
    got = single(ctx, cache, table, [n], q.cuda(), scale=scale)
    want, size, top = plain.attention(q.double().numpy(), kf, vf, ([0], [n]), float(np.float32(scale)), pos=[n - 1])
    close(got, want, size, top, EPS["bf16"], 3)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("apart", [12, 24, 32, 60, 100])
@pytest.mark.parametrize("where", ["one tile", "before", "after", "everywhere"])
def test_value_scales_far_apart(ctx, fmt, ty, apart, where):
    """Keys that weigh nearly everything hold values far smaller than those of keys that weigh next to
    nothing: 2^-(apart + 20) of them, so that theirs is all of the sum but 2^-20."""
    g = gen(46)
    n, dim = 700, 64
    v = (rn(g, n, 1, dim) * 40).round().clamp(-120, 120)
    k = torch.full((n, 1, dim), 8.0)
    small = {"one tile": torch.arange(640, 672, 3), "before": torch.arange(0, 300), "after": torch.arange(400, 700),
             "everywhere": torch.arange(0, 700, 2)}[where]
    heavy = torch.zeros(n, dtype=torch.bool)
    heavy[small] = True
    vs = (0.02 * (0.5 + torch.rand(n, 1, generator=g)))
    vs[~heavy] *= 2.0 ** apart
    # Scores: q . k = 8 * 64 ks scale; the heavy ones higher by (apart + 20) bits.
    ks = torch.full((n, 1), 1.0)
    q = torch.full((1, 4, dim), 1.0).to(TYPES[ty])
    ks[~heavy] = 1.0 - (apart + 20) / 128
    scale = 128 * float(np.log(2)) / (8 * dim)
    cache, table, kf, vf = held(ctx, fmt, k, v, ks, vs)
    got = single(ctx, cache, table, [n], q.cuda(), scale=scale)
    want, size, top = plain.attention(host(q), kf, vf, ([0], [n]), float(np.float32(scale)), pos=[n - 1])
    close(got, want, size, top, EPS[ty], 3)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("least", [2.0 ** -110, 2.0 ** -127, 2.0 ** -140, 2.0 ** -149])
def test_value_scales_past_every_span(ctx, fmt, least):
    """Scales down to float32's least beside ones: nothing beside those, in every tile."""
    g = gen(48)
    n, dim = 300, 64
    k, v = ((rn(g, n, 1, dim) * 40).round() for _ in range(2))
    ks, vs = (0.02 * (0.5 + torch.rand(n, 1, generator=g)) for _ in range(2))
    vs[::7] = least
    vs[::11] = 2.0 ** -30
    vs[::13] = 0.0
    cache, table, kf, vf = held(ctx, fmt, k, v, ks, vs)
    q = rn(g, 1, 4, dim).half()
    got = single(ctx, cache, table, [n], q.cuda())
    want, size, top = plain.attention(host(q), kf, vf, ([0], [n]), dim ** -0.5, pos=[n - 1])
    close(got, want, size, top, EPS["f16"], 3)


def test_log_sums_to_the_last_bit(ctx):
    """Rows of equal logits a block: the exponentials inside a block are ones, their sums whole, and what is left is the join
    of the blocks, in float64. The score is that sum less itself, so no other rounding hides it."""
    blocks, size = 40, 2048
    for step in (0.37, 1.7, 0.011):
        tops = -np.float32(step) * np.arange(blocks, dtype=np.float32)
        x = torch.from_numpy(np.repeat(tops, size)[None]).cuda()
        lse = float(np.log((size * np.exp(tops.astype(np.float64))).sum()))
        scores = np.full((1, 1), np.float32(lse))
        out = [torch.zeros(1, 1, device="cuda")] + [i32([[0]]) for _ in range(3)]
        sc = torch.from_numpy(scores).cuda()
        torch.cuda.synchronize()
        ocrhip.beam_select(ctx, x, sc, None, None, *out)
        ctx.synchronize()
        assert int(out[2][0, 0]) == 0
        # Forty float64 exponentials and a logarithm of numbers near ten: 2^-45; the result's own rounding 2^-24 of it.
        want = float(scores[0, 0]) - lse
        assert abs(float(out[0][0, 0]) - want) <= 2.0 ** -45 + 2.0 ** -24 * abs(want)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 40, 20])
def test_scales_and_codes_to_the_last_bit(ctx, fmt, dim):
    """A vector's scale is the float32 quotient of its largest magnitude, and a code the value's own
    rounding unless that lies within two float32 roundings of a border (2^-23 of the code): half of the values lie
    just past that, by the tiles (64, 40) and by the row (20)."""
    g = np.random.default_rng(47)
    n, most = 400, plain.QMAX[fmt]
    m = np.exp2(g.uniform(-20, 20, (n, 1))).astype(np.float32)
    codes = g.integers(0, 126, (n, dim)) + 0.5 if fmt == "i8" else (8 + g.integers(0, 8, (n, dim)) + 0.5) * 2.0 ** g.integers(-3, 5, (n, dim))
    x = (codes * (1 + g.choice([-1, 1], (n, dim)) * 2.0 ** -22.2) * m / most).astype(np.float32)
    x[:, dim // 2:] = (g.uniform(-1, 1, (n, dim - dim // 2)) * m).astype(np.float32)
    x = np.clip(x, -m, m)
    x[:, 3:4] = m
    mem = [torch.zeros(n, 1, 1, dim, dtype=torch.int8 if fmt == "i8" else torch.uint8, device="cuda") for _ in range(2)]
    mem += [torch.zeros(n, 1, 1, device="cuda") for _ in range(2)]
    cache = ocrhip.KvCache(ctx, n, 1, 1, dim, fmt, memory=mem)
    q = torch.zeros(n, 1, dim, dtype=torch.float16, device="cuda")
    table, seq, pos, xs = i32(np.arange(n)[None]), i32(np.zeros(n)), i32(np.arange(n)), torch.from_numpy(np.tile(x, (1, 3))).cuda()
    torch.cuda.synchronize()
    cache.append(table, seq, pos, xs, q, rot=0)
    ctx.synchronize()
    y = x.astype(np.float64) * most / m
    for code, scale in ((mem[0], mem[2]), (mem[1], mem[3])):
        assert np.array_equal(scale.cpu().numpy().reshape(n, 1), m / np.float32(most))
        if fmt == "i8":
            got, step = host(code).reshape(n, dim), np.ones_like(y)
        else:
            got = plain.e4m3_value(host(code)).reshape(n, dim)
            step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        want = np.rint(y / step) * step
        border = np.abs(np.abs(y / step - np.floor(y / step)) - 0.5) * step <= 2.0 ** -23 * np.abs(y)
        assert np.array_equal(got[~border], want[~border]), (np.abs(got - want)[~border] > 0).sum()


@pytest.mark.parametrize("dim", [64, 20])
def test_norms_of_constant_vectors(ctx, dim):
    """A constant vector c has sums without roundings: c / sqrt(c^2) is off by the reciprocal root's half step
    and a quarter (what corrects it is float32 too), the product's and the scale's half: 1.75 x 2^-23."""
    c = np.float32([3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37, 41, 43, 47, 53, 59, 61, 97, 101, 1.5, 0.375, 3 * 2.0 ** -40, 5 * 2.0 ** 40])
    n = len(c)
    mem = [torch.zeros(n, 1, 1, dim, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(n, 1, 1, device="cuda") for _ in range(2)]
    cache = ocrhip.KvCache(ctx, n, 1, 1, dim, "i8", memory=mem)
    q = torch.zeros(n, 1, dim, dtype=torch.float16, device="cuda")
    ones = torch.ones(dim, device="cuda")
    table, seq, pos, xs = i32(np.arange(n)[None]), i32(np.zeros(n)), i32(np.arange(n)), torch.from_numpy(np.repeat(c[:, None], 3 * dim, 1)).cuda()
    torch.cuda.synchronize()
    cache.append(table, seq, pos, xs, q, None, ones, ones, eps=0.0, rot=0)
    ctx.synchronize()
    assert (np.abs(host(mem[2]).reshape(n) * 127 - 1) <= 1.75 * 2.0 ** -23 * (1 + 2.0 ** -10)).all()
    assert (host(mem[0]) == 127).all() and (host(q) == 1).all()


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("scale,cap,size", [(1e-12, 1.0, 2.0 ** 18), (1e-6, 1e5, 2.0 ** 6), (1e-25, 1e3, 2.0 ** 40), (1e6, 1e13, 2.0 ** -10), (3e-38, 1e-3, 2.0 ** 60)])
def test_prompts_of_caps_whose_powers_are_no_floats(ctx, ty, scale, cap, size):
    """scale / cap from 10^-28 to 10^-7: scores of a third of the cap and of next to nothing."""
    if ty == "f16":
        size = min(size, 2.0 ** 9)
    g = gen(49)
    q, k, v = (rn(g, 200, h, 128) for h in (4, 2, 2))
    q, k, v = (x.to(TYPES[ty]).cuda() for x in (q * size, k * size, v))
    got = prompt(ctx, q, k, v, scale=scale, cap=cap)
    want, size, top = plain.attention(host(q), host(k), host(v), plain.key_ranges(200, None, None), float(np.float32(scale)), float(np.float32(cap)))
    close(got, want, size, min(top, cap), EPS[ty])
