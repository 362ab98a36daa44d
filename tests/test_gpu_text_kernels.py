"""The text decoder's kernels where their own choices could go wrong: every variant of a launch, ends
of tiles, values that a lower precision would lose, ties, long pools. Against float64
(oracle/text.py); tolerances as in test_gpu_text.py: half a step of a type is EPS / 2 of the value,
an attention's weights are rounded once to 16 bits (an error of the sum of p |v|), its output once
more, scores are float32 sums."""
import numpy as np
import pytest
import torch

import ocrhip
from ocrhip import text
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
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


def attend(ctx, q, k, v, docs=None, prefix=None, **kw):
    out = torch.full_like(q, 9.0)
    args = [None if x is None else i32(x) for x in (docs, prefix)]
    if kw.get("slopes") is not None:
        kw["slopes"] = torch.from_numpy(kw["slopes"]).cuda()
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, *args, **kw)
    ctx.synchronize()
    return host(out)


def some_rows(n, docs, tile):
    """Rows where something changes: documents' first and last tokens, tiles' ends, and a few others."""
    rows = {0, 1, n - 1, n // 2, n // 3}
    for d in docs:
        rows |= {d - 1, d, d + 1}
    for t in range(0, n, max(tile, n // 4 // tile * tile)):
        rows |= {t - 1, t, t + 31, t + 32, t + 63}
    return np.array(sorted(r for r in rows if 0 <= r < n))


@pytest.mark.parametrize("dim", [32, 64, 72, 96, 128, 256])
@pytest.mark.parametrize("hq,hk,lens,prefix", [
    (48, 6, [700, 1, 64, 1500], [300, 0, 64, 10]),  # many tiles: 128 queries a workgroup
    (8, 8, [900], [900]),
    (5, 1, [129, 63, 65, 0, 31], [0, 63, 0, 0, 5]),  # few: 64
])
@pytest.mark.parametrize("kind", ["plain", "capped", "bias"])
def test_attention_tiles(ctx, dim, hq, hk, lens, prefix, kind):
    g = gen(dim + hq)
    docs = 3 + np.concatenate([[0], np.cumsum(lens)])
    n = int(docs[-1]) + 40
    ty = "f16" if dim % 64 else "bf16"
    q, k, v = (rn(g, n, h, dim).to(TYPES[ty]).cuda() for h in (hq, hk, hk))
    cap = {"plain": 0.0, "capped": 30.0, "bias": 12.0}[kind]
    sl = 2.0 ** -np.arange(1, hq + 1, dtype=np.float32) if kind == "bias" else None
    got = attend(ctx, q, k, v, docs, prefix, cap=cap, slopes=sl)
    rows = some_rows(n, docs, 64)
    ranges = plain.key_ranges(n, docs, prefix)
    want, size, top = plain.attention(host(q)[rows], host(k), host(v), (ranges[0][rows], ranges[1][rows]), dim ** -0.5, cap, sl, pos=rows)
    close(got[rows], want, size, top, EPS[ty])
    assert (got[:3] == 0).all() and (got[docs[-1]:] == 0).all()


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("scale,cap", [(-0.3, 0.0), (0.0, 0.0), (1e-30, 0.0), (-0.2, 4.0), (2.0, 30.0), (0.05, 1000.0), (0.1, 1e-3), (1e3, 1e-2)])
def test_attention_scales_and_caps(ctx, ty, many, scale, cap):
    """Scores of either sign, of no size, under a cap's half and far over it."""
    g = gen(7)
    n, hq, dim = 200, 160 if many else 4, 128
    q, k, v = (rn(g, n, h, dim).to(TYPES[ty]).cuda() for h in (hq, 2, 2))
    got = attend(ctx, q, k, v, prefix=[50], scale=scale, cap=cap)
    rows, heads = np.array([0, 1, 49, 50, 51, 130, 199]), [0, 1, hq // 2, hq - 1]
    ranges = plain.key_ranges(n, None, [50])
    for h in heads:
        kv = slice(h // (hq // 2), h // (hq // 2) + 1)
        want, size, top = plain.attention(host(q)[rows, h:h + 1], host(k)[:, kv], host(v)[:, kv], (ranges[0][rows], ranges[1][rows]), scale, cap,
                                          pos=rows)
        close(got[rows, h:h + 1], want, size, top, EPS[ty])


@pytest.mark.parametrize("ty,dim,hq", [("f16", 128, 3), ("bf16", 128, 300), ("bf16", 64, 4), ("f16", 96, 2)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_attention_beside_junk(ctx, ty, dim, hq, poison):
    """Keys and values that are not numbers where nobody looks: before, after and between documents'
    reach, in the tiles that both share."""
    g = gen(13)
    lens = [70, 45, 100]
    docs = 7 + np.concatenate([[0], np.cumsum(lens)])
    n = int(docs[-1]) + 21
    q, k, v = (rn(g, n, h, dim) for h in (hq, 1, 1))
    for x in (k, v):
        x[:7], x[docs[-1]:] = poison, poison
    v[docs[2] - 1] = poison  # the second document's last token: seen by itself alone
    q, k, v = (x.to(TYPES[ty]).cuda() for x in (q, k, v))
    got = attend(ctx, q, k, v, docs, [70, 0, 20])
    ranges = plain.key_ranges(n, docs, [70, 0, 20])
    rows = np.array([r for r in some_rows(n, docs, 64) if r != docs[2] - 1])
    clean = [np.where(np.isfinite(host(x)), host(x), 0) for x in (k, v)]
    want, size, top = plain.attention(host(q)[rows][:, :3], *clean, (ranges[0][rows], ranges[1][rows]), dim ** -0.5, pos=rows)
    close(got[rows][:, :3], want, size, top, EPS[ty])
    assert not np.isfinite(got[docs[2] - 1]).any()


def test_attention_of_minus_infinity_scores(ctx):
    """A key whose every score is minus infinity weighs nothing; a query that sees only such gives zeros."""
    n, dim = 90, 64
    q = torch.ones(n, 2, dim)
    k = rn(gen(3), n, 1, dim)
    k[:5, :, 0], k[40, :, 0] = -float("inf"), -float("inf")
    v = rn(gen(4), n, 1, dim)
    q, k, v = (x.half().cuda() for x in (q, k, v))
    got = attend(ctx, q, k, v)
    with np.errstate(invalid="ignore"):
        want, size, top = plain.attention(host(q), host(k), host(v), plain.key_ranges(n, None, None), dim ** -0.5)
    close(got, want, size, top, EPS["f16"])
    assert (got[:5] == 0).all()


@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_attention_of_small_weights(ctx, ty):
    """Thousands of keys that weigh 2^-16 of the largest each: together they are a third of the sum, so
    none may be lost to float16's range."""
    n, dim = 20000, 64
    q = torch.zeros(n, 1, dim)
    q[:, :, 0] = 1.0
    k = torch.zeros(n, 1, dim)
    k[0, :, 0] = 16 * np.log(2) * 8  # scaled by 1 / 8
    v = torch.ones(n, 1, dim)
    v[0] = -1.0
    q, k, v = (x.to(TYPES[ty]).cuda() for x in (q, k, v))
    got = attend(ctx, q, k, v)[-1:]
    want, size, top = plain.attention(host(q)[-1:], host(k), host(v), ([0], [n]), 0.125, pos=[n - 1])
    close(got, want, size, top, EPS[ty])


def paged(g, fmt, hk, dim, page, lens, width=None, scales=None):
    """(cache memory, table, k, v as float64 lists, pages): random codes, scales(shape) or around a fortieth."""
    need = [-(-n // page) for n in lens]
    width = width or max(need + [1])
    pages = sum(need) + 1
    perm = torch.randperm(pages, generator=g).tolist()
    table = np.full((len(lens), width), -1, np.int32)
    for r, m in enumerate(need):
        for c in range(m):
            table[r, c] = perm.pop()
    mem, kept = [], []
    for _ in range(2):
        if fmt == "i8":
            m = torch.randint(-127, 128, (pages, hk, page, dim), generator=g, dtype=torch.int8)
            val = m.double().numpy()
        elif fmt == "e4m3":
            m = torch.randint(0, 256, (pages, hk, page, dim), generator=g, dtype=torch.uint8)
            m = torch.where((m & 127) == 127, m ^ 1, m)
            val = plain.e4m3_value(m.numpy())
        else:
            m = rn(g, pages, hk, page, dim).to(TYPES[fmt])
            val = m.double().numpy()
        s = None
        if fmt in plain.QMAX:
            s = scales((pages, hk, page)) if scales else (0.5 + torch.rand(pages, hk, page, generator=g)) * (0.02 if fmt == "i8" else 0.008)
            val = val * s.double().numpy()[..., None]
        mem.append((m.cuda(), None if s is None else s.float().cuda()))
        kept.append([np.concatenate([val[p].transpose(1, 0, 2) for p in table[r, :need[r]]])[:n] if n else np.zeros((0, hk, dim))
                     for r, n in enumerate(lens)])
    return [mem[0][0], mem[1][0], mem[0][1], mem[1][1]], table, kept[0], kept[1], pages


def decode(ctx, cache, table, lens, q, **kw):
    out = torch.full_like(q, 9.0)
    if kw.get("slopes") is not None:
        kw["slopes"] = torch.from_numpy(kw["slopes"]).cuda()
    t, n = i32(table), i32(lens)
    torch.cuda.synchronize()
    cache.attend(t, n, q, out, **kw)
    ctx.synchronize()
    return host(out)


def want_of(q, k, v, lens, scale, cap=0.0, sl=None):
    parts = [plain.attention(q[r:r + 1], k[r], v[r], ([0], [n]), scale, cap, sl, pos=[n - 1]) for r, n in enumerate(lens)]
    return np.concatenate([p[0] for p in parts]), np.concatenate([p[1] for p in parts]), max(p[2] for p in parts)


@pytest.mark.parametrize("fmt,ty", [("i8", "f16"), ("e4m3", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [64, 112, 128, 256])
def test_decode_parts(ctx, fmt, ty, dim):
    """Sequences in many parts beside ones in one and none, a table wider than any; more positions than
    are looked up at a time."""
    g = gen(dim)
    lens = [9000, 257, 0, 1, 2500]
    mem, table, k, v, pages = paged(g, fmt, 2, dim, 64, lens, 400)
    cache = ocrhip.KvCache(ctx, pages, 64, 2, dim, fmt, memory=mem)
    q = rn(g, 5, 6, dim).to(TYPES[ty]).cuda()
    sl = 2.0 ** -np.arange(3, 9, dtype=np.float32)
    for cap, slopes in ((0.0, None), (20.0, sl)):
        got = decode(ctx, cache, table, lens, q, cap=cap, slopes=slopes)
        want, size, top = want_of(host(q), k, v, lens, dim ** -0.5, cap, slopes)
        close(got, want, size, top, EPS[ty], 3)
        assert (got[2] == 0).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("span", ["tiny", "falling", "rising", "zeros"])
def test_decode_value_scales(ctx, fmt, ty, span):
    """Value scales far from one, and of every size along a sequence."""
    g = gen(21)
    dim, n = 128, 700
    mem, table, k, v, pages = paged(g, fmt, 1, dim, 16, [n])
    at = torch.zeros(pages, 1, 16)
    for i in range(n):
        at[table[0, i // 16], 0, i % 16] = i
    most = 3.0e-6 if span == "tiny" else 0.01
    s = {"tiny": torch.full_like(at, most), "falling": 0.01 * 2.0 ** (-at / 30), "rising": 0.01 * 2.0 ** ((at - n) / 30),
         "zeros": torch.where(at < 300, 0.0, 0.01)}[span].float()
    old = mem[3].cpu().double()
    mem[3] = s.cuda()
    order = [(table[0, i // 16], i % 16) for i in range(n)]
    v = [np.stack([v[0][i] / float(old[p, 0, j]) * float(s[p, 0, j]) for i, (p, j) in enumerate(order)])]
    cache = ocrhip.KvCache(ctx, pages, 16, 1, dim, fmt, memory=mem)
    q = rn(g, 1, 4, dim).to(TYPES[ty]).cuda()
    got = decode(ctx, cache, table, [n], q)
    want, size, top = want_of(host(q), k, v, [n], dim ** -0.5)
    close(got, want, size, top, EPS[ty], 3)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_decode_queries_of_any_size(ctx, fmt):
    """bfloat16 queries past float16's range, and heads of very different size beside each other."""
    g = gen(22)
    dim, lens = 64, [300, 40]
    mem, table, k, v, pages = paged(g, fmt, 1, dim, 16, lens)
    cache = ocrhip.KvCache(ctx, pages, 16, 1, dim, fmt, memory=mem)
    q = rn(g, 2, 4, dim)
    q[:, 0] *= 1e6
    q[:, 1] *= 3e4
    q[1, 2] = 0
    q = q.bfloat16().cuda()
    got = decode(ctx, cache, table, lens, q, scale=1e-6)
    want, size, top = want_of(host(q), k, v, lens, 1e-6)
    close(got, want, size, top, EPS["bf16"], 3)


def test_decode_of_what_is_not_a_number(ctx):
    """A vector that reads as NaN spoils its own sequence and head, also over a part's end; junk past a
    length spoils nothing."""
    g = gen(23)
    dim, lens = 64, [600, 600, 33]
    mem, table, k, v, pages = paged(g, "i8", 2, dim, 16, lens)
    mem[3][table[0, 5], 1, 3] = float("nan")
    last = table[2, 2]
    mem[2][last, :, 1:], mem[3][last, :, 1:] = float("nan"), float("nan")
    cache = ocrhip.KvCache(ctx, pages, 16, 2, dim, "i8", memory=mem)
    q = rn(g, 3, 4, dim).half().cuda()
    got = decode(ctx, cache, table, lens, q)
    want, size, top = want_of(host(q), k, v, lens, dim ** -0.5)
    assert np.isnan(got[0, 2:]).all()
    fine = np.ones(got.shape, bool)
    fine[0, 2:] = False
    close(got[fine], want[fine], size[fine], top, EPS["f16"], 3)


def test_largest_bfloat16_values(ctx):
    """Values near the type's largest: their weighted means are, the sums on the way must be."""
    g = gen(25)
    n, dim, page = 120, 64, 16
    q, k = (rn(g, n, h, dim).bfloat16().cuda() for h in (4, 1))
    v = ((0.5 + 0.4 * torch.rand(n, 1, dim, generator=g)) * 3.3e38 / n).bfloat16()
    v[:60] = -v[:60]
    v = v.cuda()
    got = attend(ctx, q, k, v)
    want, size, top = plain.attention(host(q), host(k), host(v), plain.key_ranges(n, None, None), dim ** -0.5)
    close(got / 1e36, want / 1e36, size / 1e36, top, EPS["bf16"])
    pages = -(-n // page)
    mem = [torch.zeros(pages, 1, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [None, None]
    for m, x in zip(mem, (k, v)):
        m.view(-1, dim)[:n] = x[:, 0]
    cache = ocrhip.KvCache(ctx, pages, page, 1, dim, "bf16", memory=mem)
    got = decode(ctx, cache, [list(range(pages))], [n], q[-1:])
    close(got / 1e36, want[-1:] / 1e36, size[-1:] / 1e36, top, EPS["bf16"], 3)


def test_read_past_a_grid(ctx):
    """More pieces of sequences than a launch has workgroups."""
    rows, most, dim = 2 ** 22 + 5, 3, 8
    mem = [torch.arange(2 * 4 * dim, dtype=torch.float32).view(2, 1, 4, dim).half().cuda() for _ in range(2)] + [None, None]
    cache = ocrhip.KvCache(ctx, 2, 4, 1, dim, "f16", memory=mem)
    table = (torch.arange(rows, device="cuda", dtype=torch.int32) % 2)[:, None].contiguous()
    lens = torch.full((rows,), 2, dtype=torch.int32, device="cuda")
    k, v = (torch.full((rows, most, 1, dim), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.read(table, lens, k, v)
    ctx.synchronize()
    want = torch.cat([mem[0][:, 0, :2], torch.zeros(2, 1, dim, device="cuda", dtype=torch.float16)], 1)[table[:, 0].long()]
    assert torch.equal(k[:, :, 0], want) and torch.equal(v, k)


@pytest.mark.parametrize("fmt", ["i8", "f16"])
def test_pools_past_32_bits(ctx, fmt):
    """Vectors whose first byte is more than 2^32 into the pool: written, read and attended to."""
    g = gen(24)
    hk, page, dim = 8, 64, 128
    per = hk * page * dim * (1 if fmt == "i8" else 2)
    pages = 2 ** 32 // per + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * per + (1 << 30):
        pytest.skip("not enough memory")
    ty = torch.int8 if fmt == "i8" else torch.float16
    mem = [torch.empty(pages, hk, page, dim, dtype=ty, device="cuda") for _ in range(2)]
    mem += [torch.empty(pages, hk, page, device="cuda") for _ in range(2)] if fmt == "i8" else [None, None]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    n = 150
    table = np.array([[pages - 1, 3, pages - 20]], np.int32)
    x = rn(g, n, 3 * hk * dim).half().cuda()
    q = torch.zeros(n, hk, dim, dtype=torch.float16, device="cuda")
    ko, vo = (torch.zeros(1, n, hk, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    out = torch.zeros(1, hk, dim, dtype=torch.float16, device="cuda")
    t, seq, pos, lens = i32(table), i32([0] * n), i32(range(n)), i32([n])
    torch.cuda.synchronize()
    cache.append(t, seq, pos, x, q, rot=0)
    cache.read(t, lens, ko, vo)
    cache.attend(t, lens, q[-1:], out)
    ctx.synchronize()
    _, k, v = plain.projections(host(x), hk, hk, dim, np.arange(n), None, None, 1e-6, 0, 1e4, "halves")
    for got, want in ((host(ko)[0], k), (host(vo)[0], v)):
        tol = plain.half_step(want, fmt) * (1 + 2.0 ** -10) + 2.0 ** -10 * np.abs(want) if fmt == "i8" else 0 * want
        assert (np.abs(got - want) <= tol + 2.0 ** -18 * np.abs(want).max(-1, keepdims=True)).all()
    want, size, top = plain.attention(host(q)[-1:], host(ko)[0], host(vo)[0], ([0], [n]), dim ** -0.5, pos=[n - 1])
    # The values read back were rounded to float16 once more.
    close(host(out), want, size, top, EPS["f16"], 4)


@pytest.mark.parametrize("dim,rot,pairs", [(8, 8, "halves"), (24, 8, "adjacent"), (40, 24, "halves"), (104, 4, "adjacent"), (136, 128, "halves"), (256, 200, "halves"),
                                           (64, 36, "halves")])
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f16"])
@pytest.mark.parametrize("n", [5, 4099])
def test_append_shapes(ctx, dim, rot, pairs, fmt, n):
    """Vectors of any number of eights, rotations that end inside one, tokens for four of a workgroup
    and some over, projections that lie on no more than their type's size."""
    g = gen(dim + n)
    hq, hk, page = 3, 1, 32
    width = (hq + 2 * hk) * dim
    flat = rn(g, n * (width + 1) + 1).half().cuda()
    x = flat[1:].view(n, width + 1)[:, :width]
    pages = -(-n // page)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].cuda().contiguous()
    ty = {"i8": torch.int8, "e4m3": torch.uint8, "f16": torch.float16}[fmt]
    mem = [torch.zeros(pages, hk, page, dim, dtype=ty, device="cuda") for _ in range(2)]
    mem += [torch.zeros(pages, hk, page, device="cuda") for _ in range(2)] if fmt != "f16" else [None, None]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    norms = [1 + 0.3 * rn(g, dim) for _ in range(2)]
    q, k = torch.zeros(n, hq, dim, dtype=torch.float16, device="cuda"), torch.zeros(n, hk, dim, dtype=torch.float16, device="cuda")
    pos = torch.randperm(n, generator=g)
    args = [table, i32([0] * n), pos.to(torch.int32).cuda(), x, q, k] + [w.cuda() for w in norms]
    ko, vo = (torch.zeros(1, n, hk, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.append(*args, rot=rot, pairs=pairs)
    cache.read(table, i32([n]), ko, vo)
    ctx.synchronize()
    eq, ek, ev = plain.projections(host(x), hq, hk, dim, pos.numpy(), *[w.double().numpy() for w in norms], 1e-6, rot, 1e4, pairs)
    for got, want in ((q, eq), (k, ek)):
        top = np.abs(want).max(-1, keepdims=True)
        assert (np.abs(host(got) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * top + 2.0 ** -24).all()
    for got, want in ((host(ko)[0][pos], ek), (host(vo)[0][pos], ev)):
        top = np.abs(want).max(-1, keepdims=True)
        tol = 2.0 ** -10 * np.abs(want) + 2.0 ** -18 * top + 2.0 ** -24
        if fmt != "f16":
            tol = tol + plain.half_step(want, fmt) * (1 + 2.0 ** -10)
        assert (np.abs(got - want) <= tol).all()


def beam(ctx, x, scores, finished, eos):
    g, w = scores.shape
    out = [torch.zeros(g, w, device="cuda")] + [i32(np.full((g, w), -5)) for _ in range(3)]
    sc, fin = torch.from_numpy(scores.astype(np.float32)).cuda(), None if finished is None else i32(finished)
    torch.cuda.synchronize()
    ocrhip.beam_select(ctx, x, sc, fin, eos, *out)
    ctx.synchronize()
    want = plain.beam_select(host(x), scores.astype(np.float32), finished, -1 if eos is None else eos)
    got = [host(o) for o in out]
    for a, b in zip(got[1:], want[1:]):
        assert np.array_equal(a, b), (a, b)
    fine = np.isfinite(want[0])
    assert np.array_equal(got[0][~fine], want[0][~fine])
    assert (np.abs(got[0][fine] - want[0][fine]) <= 2.0 ** -24 * np.abs(want[0][fine]) + 2.0 ** -21).all()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [2048, 2049, 4097, 131073, 300001, 1500000])
def test_beam_vocabularies(ctx, ty, vocab):
    """Rows of one block and of several chunks a block, with ends inside a part; rows that lie on no
    more than their type's size."""
    g = gen(vocab)
    x = (rn(g, 4 * (vocab + 1) + 1) * 3).to(TYPES[ty]).cuda()[1:].view(4, vocab + 1)[:, :vocab]
    beam(ctx, x, -5 * torch.rand(2, 2, generator=g).numpy(), None, 1)
    x[:, vocab - 3:] = 20.0  # the best at the very end
    beam(ctx, x, -5 * torch.rand(1, 4, generator=g).numpy(), None, None)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [97, 2000, 100000])
@pytest.mark.parametrize("w", [1, 5, 32])
def test_beam_ties_and_orders(ctx, ty, vocab, w):
    """All alike; a handful that count among minus infinities; rising and falling rows, whose best share
    a part; many that share the threshold; NaN among them."""
    g = gen(vocab + w)
    up = torch.arange(vocab).float()
    rows = [torch.zeros(vocab), torch.full((vocab,), -float("inf")).index_fill(0, torch.randint(0, vocab, (7,), generator=g), 1.0), up / vocab,
            -up / vocab, torch.where(rn(g, vocab) > 1.5, 4.0, -1.0), torch.where(rn(g, vocab) > 0, float("nan"), 2.0), (up % 100 == 3).float(),
            torch.where(up < 600, 3.0, up.sin())]
    for k in range(0, 8, 4):
        x = torch.stack([rows[(k + i) % 8] for i in range(4)])
        x = x.repeat_interleave(w, 0).to(TYPES[ty]).cuda()
        scores = np.tile(-np.arange(w, dtype=np.float64) * 0.75, (4, 1))
        beam(ctx, x, scores, None, None)
        beam(ctx, x, scores, (torch.rand(4, w, generator=g) < 0.5).int().numpy(), min(2, vocab - 1))


def test_the_same_twice(ctx):
    """Nothing depends on the order in which workgroups run."""
    g = gen(31)
    lens = [3000, 100, 1700]
    mem, table, *_, pages = paged(g, "i8", 2, 128, 16, lens)
    cache = ocrhip.KvCache(ctx, pages, 16, 2, 128, "i8", memory=mem)
    q = rn(g, 3, 8, 128).bfloat16().cuda()
    a = [decode(ctx, cache, table, lens, q) for _ in range(3)]
    x = [rn(g, 1000, h, 128).bfloat16().cuda() for h in (8, 2, 2)]
    b = [attend(ctx, *x) for _ in range(3)]
    for y in (a, b):
        assert np.array_equal(y[0], y[1]) and np.array_equal(y[0], y[2])


def test_both_ways_to_the_library(ctx, monkeypatch):
    """Calls on tensors by the native module and by the binding's own checks do the same."""
    g = gen(32)
    dim, page, hq, hk, n = 64, 16, 4, 2, 40
    x = rn(g, n, (hq + 2 * hk) * dim).half().cuda()
    logits = rn(g, 6, 5000).cuda()
    norm = 1 + 0.1 * rn(g, dim).cuda()
    res = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(text, "_native", lambda *a: False)
        mem = [torch.zeros(8, hk, page, dim, dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.zeros(8, hk, page, device="cuda") for _ in range(2)]
        cache = ocrhip.KvCache(ctx, 8, page, hk, dim, "e4m3", memory=mem)
        t, pos, lens = i32([[4, 1, 6]]), i32(range(n)), i32([n])
        q, k = torch.zeros(n, hq, dim, dtype=torch.float16, device="cuda"), torch.zeros(n, hk, dim, dtype=torch.float16, device="cuda")
        o, one = torch.zeros_like(q), torch.zeros(1, hq, dim, dtype=torch.float16, device="cuda")
        ko, vo = (torch.zeros(1, 50, hk, dim, dtype=torch.float16, device="cuda") for _ in range(2))
        sc, par, tok, fin = torch.zeros(2, 3, device="cuda"), *(i32(np.zeros((2, 3))) for _ in range(3))
        t2, l2, u2 = i32(np.zeros((1, 3))), i32([0]), i32([0])
        sl = torch.tensor([0.5, 0.25, 0.125, 0.0625]).cuda()
        torch.cuda.synchronize()
        cache.append(t, i32([0] * n), pos, x, q, k, norm, norm, rot=32, pairs="adjacent")
        cache.read(t, lens, ko, vo)
        cache.attend(t, lens, q[-1:], one, cap=5.0, slopes=sl)
        ocrhip.attention(ctx, q, k, x[:, (hq + hk) * dim:].unflatten(1, (hk, dim)), o, i32([0, n]), i32([7]), slopes=sl)
        ocrhip.beam_select(ctx, logits, torch.zeros(2, 3, device="cuda"), None, None, sc, par, tok, fin)
        cache.fork(t, lens, i32([[0]]), i32([7]), t2, l2, u2)
        ctx.synchronize()
        res.append([y.clone() for y in (*mem, q, k, o, one, ko, vo, sc, par, tok, fin, t2, l2, u2)])
        assert float(one.abs().sum()) > 0 and float(o.abs().sum()) > 0 and float(ko.abs().sum()) > 0
    for a, b in zip(*res):
        assert torch.equal(a, b)
    monkeypatch.undo()
    for bad in (x[:, :-1], x.cpu(), x.double(), x[:-1]):
        with pytest.raises(ocrhip.OcrError):
            cache.append(t, i32([0] * n), pos, bad, q)
    with pytest.raises(ocrhip.OcrError, match="scale"):
        ocrhip.attention(ctx, q, k, k, o, scale=float("nan"))
