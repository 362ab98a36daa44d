"""Rotary positions of several axes on the GPU against float64 (oracle/text.py): alone and in the cache's append.

An output is rounded once, half a step of its type; turns and products are float32: 2^-20 of the pair's length."""
import numpy as np
import pytest
import torch

import ocrhip
from oracle import text as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rn(g, *shape):
    return torch.randn(*shape, generator=g)


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to("cuda")


def host(x):
    torch.cuda.synchronize()
    return x.cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()


def close(got, want, ty):
    top = np.abs(want).max(-1, keepdims=True) if want.size else 0
    bad = np.abs(got - want) > EPS[ty] / 2 * np.abs(want) + 2.0 ** -20 * top + (2.0 ** -24 if ty == "f16" else 0)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


ROTATE = [
    # type, heads, dim, first, rot, pairs, axes, order, ladder
    ("f16", 2, 64, 0, 64, "halves", (16, 8, 8), "blocks", "shared"),
    ("bf16", 16, 80, 0, 80, "halves", (20, 20), "blocks", "own"),
    ("bf16", 3, 128, 0, 128, "adjacent", (24, 20, 20), "turns", "shared"),
    ("f32", 1, 96, 32, 64, "halves", (5, 9, 10, 8), "turns", "own"),
    ("f16", 5, 192, 128, 64, "adjacent", (32,), "blocks", "shared"),
    ("f32", 2, 15, 3, 6, "halves", (1, 2), "turns", "own"),
    ("bf16", 4, 40, 4, 24, "adjacent", (0, 12), "blocks", "own"),
    ("f16", 1, 2, 0, 2, "halves", (0, 1, 0), "turns", "shared"),
    ("f32", 2, 64, 8, 0, "halves", (0,), "blocks", "shared"),
    ("bf16", 7, 256, 0, 256, "halves", (128,), "blocks", "shared"),
    ("f16", 2, 1024, 512, 256, "halves", (60, 68), "turns", "shared"),
    ("bf16", 130, 64, 0, 32, "halves", (6, 5, 5), "turns", "own"),
]


@pytest.mark.parametrize("ty,heads,dim,first,rot,pairs,axes,order,ladder", ROTATE)
@pytest.mark.parametrize("n,layout", [(1, "apart"), (37, "packed"), (37, "place"), (261, "odd"), (5, "back")])
def test_rotate(ctx, ty, heads, dim, first, rot, pairs, axes, order, ladder, n, layout):
    g = gen(n + dim + rot)
    off, pad = (1, 3) if layout == "odd" else (0, 0)
    wide = (2 * heads * dim + pad) if layout != "apart" else heads * dim
    flat = rn(g, n * wide + off).to(TYPES[ty]).cuda()
    x = flat[off:].view(n, wide)[:, : heads * dim].unflatten(1, (heads, dim))
    if layout == "odd" and heads > 1:  # heads apart as well
        x = flat[off:].view(n, wide)[:, : 2 * heads * dim].unflatten(1, (heads, 2 * dim))[..., :dim]
    at = torch.randint(0, 2000000, (n, len(axes)), generator=g).to(torch.int32)
    at[0] = -5  # a position before the start turns the other way
    want = plain.rotate_axes(host(x), at.numpy(), first, rot, 1e4, pairs, axes, order, ladder, layout == "back")
    before = flat.clone()
    out = None if layout == "place" else torch.full((n, heads, dim), 9.0, dtype=TYPES[ty], device="cuda")
    args = at.cuda()
    torch.cuda.synchronize()
    ocrhip.rotate(ctx, x, args, out, first=first, rot=rot, theta=1e4, pairs=pairs, axes=axes, order=order, ladder=ladder, back=layout == "back")
    ctx.synchronize()
    close(host(x if out is None else out), want, ty)
    if out is not None:
        assert torch.equal(flat.cpu(), before.cpu())
    else:  # what lies between the vectors stays
        changed = (flat != before).cpu()[off:].view(n, wide)
        assert not changed[:, heads * dim:].any()


def test_back_is_the_gradient(ctx):
    """The rotation is linear: against the transposed rotation, and against differences of <rotate(x), g>."""
    g = gen(3)
    n, heads, dim, axes = 4, 2, 16, (3, 5)
    x, up = rn(g, n, heads, dim).cuda(), rn(g, n, heads, dim).cuda()
    at = torch.randint(0, 500, (n, 2), generator=g).to(torch.int32).cuda()
    kw = dict(axes=axes, order="turns", ladder="own", theta=100.0)
    grad, y, back = (torch.empty_like(x) for _ in range(3))
    torch.cuda.synchronize()
    ocrhip.rotate(ctx, up, at, grad, back=True, **kw)
    ocrhip.rotate(ctx, x, at, y, **kw)
    ocrhip.rotate(ctx, y, at, back, back=True, **kw)
    ctx.synchronize()
    f = lambda v: (plain.rotate_axes(v, at.cpu().numpy(), 0, dim, 100.0, "halves", axes, "turns", "own") * host(up)).sum()  # noqa: E731
    xs = host(x)
    for place in [(0, 0, 0), (1, 1, 7), (2, 0, 8), (3, 1, 15)]:
        step = np.zeros_like(xs)
        step[place] = 0.5
        assert abs((f(xs + step) - f(xs - step)) - host(grad)[place]) <= 2.0 ** -20 * 8
    assert np.abs(host(back) - xs).max() <= 2.0 ** -20 * np.abs(xs).max() * 2


@pytest.mark.parametrize("tin,tout,fmt,hq,hk,dim,rot,pairs,axes,order,ladder", [
    ("bf16", "bf16", "bf16", 4, 2, 128, 128, "halves", (24, 20, 20), "turns", "shared"),
    ("f32", "f16", "f16", 2, 1, 64, 32, "adjacent", (8, 8), "blocks", "own"),
    ("f16", "f16", "f16", 3, 3, 15, 14, "halves", (3, 2, 2), "turns", "own"),
    ("bf16", "bf16", "i8", 8, 1, 80, 80, "halves", (10, 10, 20), "blocks", "shared"),
])
@pytest.mark.parametrize("n", [1, 9, 5000])
def test_append(ctx, tin, tout, fmt, hq, hk, dim, rot, pairs, axes, order, ladder, n):
    """Tokens go where pos says, turned by at."""
    if n == 5000 and dim == 15:
        n = 300
    g = gen(n + dim)
    page = 16
    pages = -(-n // page)
    shape = (pages, hk, page, dim)
    mem = [torch.zeros(shape, dtype=torch.int8 if fmt == "i8" else TYPES[fmt], device="cuda") for _ in range(2)]
    mem += [torch.zeros(shape[:3], device="cuda") for _ in range(2)] if fmt == "i8" else [None, None]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    x = rn(g, n, (hq + 2 * hk) * dim).to(TYPES[tin]).cuda()
    at = torch.randint(0, 100000, (n, len(axes)), generator=g).to(torch.int32)
    q, k = (torch.full((n, h, dim), 9.0, dtype=TYPES[tout], device="cuda") for h in (hq, hk))
    norm = (1 + 0.2 * rn(g, dim)).cuda()
    table, seq, pos, ats = i32(torch.randperm(pages, generator=g)[None]), i32([0] * n), i32(range(n)), at.cuda()
    torch.cuda.synchronize()
    cache.append(table, seq, pos, x, q, k, norm, norm, eps=1e-5, rot=rot, theta=5e5, pairs=pairs, at=ats, axes=axes, order=order, ladder=ladder)
    ctx.synchronize()
    y = host(x).reshape(n, hq + 2 * hk, dim)
    wn = host(norm)
    turn = lambda v: plain.rotate_axes(plain.norm(v, wn, 1e-5), at.numpy(), 0, rot, 5e5, pairs, axes, order, ladder)  # noqa: E731
    wq, wk = turn(y[:, :hq]), turn(y[:, hq: hq + hk])
    close(host(q), wq, tout)
    close(host(k), wk, tout)
    if fmt != "i8":
        held = host(mem[0])[host(table)[0]].transpose(0, 2, 1, 3).reshape(-1, hk, dim)[:n]
        assert np.array_equal(held, host(k))  # the same rounding
    else:
        held = (host(mem[0]) * host(mem[2])[..., None])[host(table)[0]].transpose(0, 2, 1, 3).reshape(-1, hk, dim)[:n]
        assert (np.abs(held - wk) <= plain.half_step(wk, "i8") * 1.001 + 2.0 ** -20 * np.abs(wk).max(-1, keepdims=True)).all()


def test_one_axis_is_the_token_position(ctx):
    """An axis that has all pairs gives what the call without axes gives, bit by bit."""
    g = gen(5)
    n, hq, hk, dim = 70, 4, 2, 64
    x = rn(g, n, (hq + 2 * hk) * dim).to(torch.bfloat16).cuda()
    cache = ocrhip.KvCache(ctx, 8, 16, hk, dim, "bf16")
    table, seq, pos = i32([range(8)]), i32([0] * n), i32(range(n))
    outs = [[torch.zeros(n, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, hk)] for _ in range(3)]
    torch.cuda.synchronize()
    cache.append(table, seq, pos, x, *outs[0])
    cache.append(table, seq, pos, x, *outs[1], at=pos)
    cache.append(table, seq, pos, x, *outs[2], at=pos[:, None].contiguous(), axes=(32,), order="turns", ladder="own")
    ctx.synchronize()
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


def test_no_tokens(ctx):
    x = torch.zeros(0, 2, 8, device="cuda")
    ocrhip.rotate(ctx, x, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), axes=(2, 2))
    ctx.synchronize()
