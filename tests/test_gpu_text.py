"""The text decoder's operators on the GPU against float64 (oracle/text.py).

Tolerances count roundings: half a step of a type is EPS / 2 of the value. An attention's weights are
rounded once to the 16-bit type, and so are the values an 8-bit cache stands for: both are errors of the sum of p |v|;
the output is rounded once more. Scores are float32 sums: an error of 2^-21 of the largest, which the exponential
passes on to the weights, and exp and tanh themselves are good to 2^-20."""
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


def dev(x, dtype=None):
    return x.to(dtype).to("cuda") if dtype else x.to("cuda")


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to("cuda")


def host(x):
    torch.cuda.synchronize()
    return x.cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()


def cache_memory(g, pages, heads, page, dim, fmt, junk=True):
    """A cache full of values (junk: NaN or what the scale makes of it) that no test may read."""
    shape = (pages, heads, page, dim)
    scales = [None, None]
    if fmt == "i8":
        mem = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)]
    elif fmt == "e4m3":
        mem = [torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2)]
    else:
        mem = [torch.full(shape, float("nan") if junk else 0.0).to(TYPES[fmt]) for _ in range(2)]
    if fmt in plain.QMAX:
        scales = [torch.full(shape[:3], float("nan")).cuda() for _ in range(2)]
    torch.cuda.synchronize()
    return [m.cuda() for m in mem] + scales


def tables(g, lens, page, width=None, spare=3):
    need = [-(-n // page) for n in lens]
    width = width or max(need + [1])
    perm = torch.randperm(sum(need) + spare, generator=g).tolist()
    t = np.full((len(lens), width), -1, np.int32)
    for r, n in enumerate(need):
        for c in range(n):
            t[r, c] = perm.pop()
    return t, sum(need) + spare, perm


APPEND = [
    # tokens' sequences and positions, types, heads, dim, rot, pairs, page
    ("f32", "f16", "f16", 2, 1, 64, 64, "halves", 16),
    ("bf16", "bf16", "i8", 8, 2, 128, 128, "halves", 16),
    ("bf16", "bf16", "e4m3", 4, 4, 128, 64, "adjacent", 64),
    ("f16", "f16", "i8", 6, 3, 80, 80, "halves", 32),
    ("f16", "f16", "e4m3", 3, 1, 96, 0, "halves", 16),
    ("f32", "bf16", "bf16", 2, 2, 256, 256, "adjacent", 16),
    ("f32", "f16", "i8", 2, 1, 15, 14, "halves", 7),
    ("bf16", "f16", "e4m3", 5, 5, 200, 2, "adjacent", 33),
    ("f16", "f16", "f16", 1, 1, 1, 0, "halves", 1),
    ("bf16", "bf16", "i8", 16, 2, 32, 32, "adjacent", 16),
    ("f32", "bf16", "e4m3", 4, 2, 72, 48, "halves", 16),
]


@pytest.mark.parametrize("tin,tout,fmt,hq,hk,dim,rot,pairs,page", APPEND)
@pytest.mark.parametrize("new", ["step", "prompt"])
def test_append_and_read(ctx, tin, tout, fmt, hq, hk, dim, rot, pairs, page, new):
    g = gen(dim + page)
    if new == "step":
        lens = [1, 5, 2 * page, 2 * page + 1, 77]
        seq, pos = list(range(5)), [n - 1 for n in lens]
    else:
        lens = [130, 1, 3 * page, 0]
        seq = [s for s, n in enumerate(lens) for _ in range(n)]
        pos = [p for n in lens for p in range(n)]
        order = torch.randperm(len(seq), generator=g).tolist()
        seq, pos = [seq[i] for i in order], [pos[i] for i in order]
    table, pages, _ = tables(g, lens, page)
    n, width = len(seq), (hq + 2 * hk) * dim
    pad = 3 if dim % 2 else 8
    wide = rn(g, n, width + pad) * (0.2 + rn(g, 1, width + pad).abs())
    norms = [None, None] if dim == 96 else [1 + 0.3 * rn(g, dim) for _ in range(2)]
    x = dev(wide, TYPES[tin])[:, :width]
    mem = cache_memory(g, pages, hk, page, dim, fmt)
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    q = torch.full((n, hq, dim), 9.0, dtype=TYPES[tout], device="cuda")
    k = torch.full((n, hk, dim), 9.0, dtype=TYPES[tout], device="cuda")
    args = [i32(table), i32(seq), i32(pos), x, q, k] + [None if w is None else dev(w) for w in norms]
    torch.cuda.synchronize()
    cache.append(*args, eps=1e-5, rot=rot, theta=5e5, pairs=pairs)
    ctx.synchronize()
    wn = [None if w is None else w.double().numpy() for w in norms]
    eq, ek, ev = plain.projections(host(x), hq, hk, dim, np.asarray(pos), *wn, 1e-5, rot, 5e5, pairs)
    half = EPS[tout] / 2
    tiny = 2.0 ** -24  # float16's smallest step
    for got, want in ((q, eq), (k, ek)):
        top = np.abs(want).max(-1, keepdims=True)  # norms and turns are float32: 2^-20 of the vector's largest
        assert (np.abs(host(got) - want) <= half * np.abs(want) + 2.0 ** -20 * top + tiny).all()
    most = max(lens) + 3
    ko, vo = (torch.full((len(lens), most, hk, dim), 9.0, dtype=TYPES[tout], device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.read(i32(table), i32(lens), ko, vo)
    ctx.synchronize()
    for got, want in ((host(ko), ek), (host(vo), ev)):
        at = got[seq, pos]
        top = np.abs(want).max(-1, keepdims=True)
        if fmt in plain.QMAX:
            # Half a code's step (a value on the border may fall either way: its own float32 error), then the output's.
            tol = plain.half_step(want, fmt) * (1 + 2.0 ** -10) + 2.0 ** -18 * top + half * np.abs(want) * (1 + 2.0 ** -3) + tiny
        else:
            tol = (EPS[fmt] / 2 + half) * np.abs(want) + 2.0 ** -20 * top + tiny
        assert (np.abs(at - want) <= tol).all()
        for s, m in enumerate(lens):
            assert (got[s, m:] == 0).all()


def test_append_drops_what_has_no_place(ctx):
    """Sequences outside the table, positions outside its pages and page numbers outside the pool
    are dropped: nothing else in the pool changes; the queries are there all the same."""
    g = gen(5)
    hq, hk, dim, page, pages = 2, 1, 64, 16, 6
    table = np.array([[2, -1], [9, 4], [-7, 6]], np.int32)
    seq = [0, 0, 0, 0, 1, 1, -1, 3, 2, 2, 0]
    pos = [3, 16, 32, -1, 0, 31, 0, 0, 0, 16, 2000000000]
    x = rn(g, len(seq), (hq + 2 * hk) * dim)
    mem = [torch.full((pages, hk, page, dim), 5, dtype=torch.int8, device="cuda") for _ in range(2)]
    mem += [torch.full((pages, hk, page), 0.5, device="cuda") for _ in range(2)]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, "i8", memory=mem)
    q = torch.zeros(len(seq), hq, dim, dtype=torch.float16, device="cuda")
    xs = dev(x)
    torch.cuda.synchronize()
    cache.append(i32(table), i32(seq), i32(pos), xs, q, rot=0)
    ctx.synchronize()
    changed = (host(mem[2]) != 0.5)
    assert changed.sum() == 2 and changed[2, 0, 3] and changed[4, 0, 15]
    for m in mem[:2]:
        rows = (host(m) != 5).any(-1)
        assert (rows == changed).all()
    assert (np.abs(host(q) - x.double().numpy()[:, : hq * dim].reshape(-1, hq, dim)) <= 2.0 ** -10).all()
    ko, vo = (torch.full((3, 35, hk, dim), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.read(i32(table), i32([32, -4, 2000000000]), ko, vo)
    ctx.synchronize()
    got = host(ko)
    assert (got[0, 16:] == 0).all() and (got[1] == 0).all() and (got[2] == 0).all() and (got[0, 4:16] == 2.5).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_vectors_of_zeros_and_infinities(ctx, fmt):
    dim, page = 64, 16
    x = torch.zeros(6, 3 * dim)
    x[1] = 1e-35
    x[2, dim + 3] = float("inf")
    x[3, 2 * dim + 5] = float("nan")
    x[4] = 3.0e38
    x[5, dim:] = torch.cat([torch.linspace(-448, 448, dim)] * 2)
    mem = cache_memory(gen(1), 2, 1, page, dim, fmt)
    cache = ocrhip.KvCache(ctx, 2, page, 1, dim, fmt, memory=mem)
    q = torch.zeros(6, 1, dim, dtype=torch.bfloat16, device="cuda")
    table, xs = i32([[1]]), dev(x)
    ko, vo = (torch.zeros(1, 6, 1, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.append(table, i32([0] * 6), i32(range(6)), xs, q, rot=0)
    cache.read(table, i32([6]), ko, vo)
    ctx.synchronize()
    k, v = host(ko)[0, :, 0], host(vo)[0, :, 0]
    assert (k[:2] == 0).all() and (v[:2] == 0).all()
    assert np.isnan(k[2]).all() and (v[2] == 0).all() and (k[3] == 0).all() and np.isnan(v[3]).all()
    assert (np.abs(k[4] / 3.0e38 - 1) <= 2.0 ** -7).all()
    want = x[5, dim: 2 * dim].double().numpy()
    assert (np.abs(k[5] - want) <= plain.half_step(want, fmt) * 1.001 + 2.0 ** -8 * np.abs(want) * 1.1).all()


@pytest.mark.parametrize("rot,pairs", [(64, "halves"), (64, "adjacent")])
def test_far_positions(ctx, rot, pairs):
    """Angles at positions up to two million are those of float64."""
    pos = [0, 1, 4095, 65537, 1000003, 2097151]
    g = gen(3)
    x = rn(g, len(pos), 3 * 64)
    mem = cache_memory(g, 1, 1, 16, 64, "f16")
    cache = ocrhip.KvCache(ctx, 1, 16, 1, 64, "f16", memory=mem)
    q = torch.zeros(len(pos), 1, 64, dtype=torch.float16, device="cuda")
    table, xs = i32(np.full((1, 131072), -1)), dev(x)
    torch.cuda.synchronize()
    cache.append(table, i32([0] * len(pos)), i32(pos), xs, q, rot=rot, theta=1e4, pairs=pairs)
    ctx.synchronize()
    want = plain.rotate(x.double().numpy().reshape(len(pos), 3, 64)[:, :1], np.asarray(pos), rot, 1e4, pairs)
    assert (np.abs(host(q) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * np.abs(want).max() + 2.0 ** -24).all()


def attention_close(got, want, size, top, eps, roundings=2):
    tol = (roundings * eps / 2 + 2.0 ** -18 + 2.0 ** -20 * top) * size + eps / 2 * np.abs(want) * (1 + eps) + 2.0 ** -24
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


ATTENTION = [
    # type, heads, dim, documents, prefix, cap, slopes
    ("f16", 2, 2, 64, [1], None, 0.0, False),
    ("bf16", 4, 1, 64, [109], [109], 0.0, False),
    ("bf16", 4, 2, 128, [17, 1, 0, 64, 129], [3, 1, 0, 64, 500], 0.0, True),
    ("f16", 2, 1, 128, [300], [77], 20.0, False),
    ("f16", 3, 3, 32, [31, 33, 200], None, 0.0, True),
    ("bf16", 8, 1, 80, [513], [512], 50.0, True),
    ("f16", 6, 2, 96, [63, 65, 127], [10, 0, 127], 5.0, True),
    ("bf16", 2, 2, 256, [150], [40], 0.0, False),
    ("f16", 2, 1, 15, [140], [20], 0.0, True),
    ("f16", 1, 1, 1, [70], None, 0.0, False),
    ("bf16", 2, 1, 8, [5, 90], None, 30.0, False),
    ("bf16", 1, 1, 128, [1100], [100], 0.0, False),
    ("f16", 16, 2, 64, [700, 1, 500], [650, 0, 0], 0.0, False),
    ("f16", 2, 2, 200, [90, 40], [0, 40], 8.0, True),
]


@pytest.mark.parametrize("ty,hq,hk,dim,lens,prefix,cap,bias", ATTENTION)
@pytest.mark.parametrize("layout", ["apart", "fused", "odd"])
def test_attention(ctx, ty, hq, hk, dim, lens, prefix, cap, bias, layout):
    g = gen(sum(lens) + dim)
    before, after = (0, 0) if len(lens) == 1 and layout == "apart" else (5, 9)
    n = sum(lens) + before + after
    docs = before + np.concatenate([[0], np.cumsum(lens)])
    t = TYPES[ty]
    if layout == "apart":
        q, k, v = (dev(rn(g, n, h, dim), t) for h in (hq, hk, hk))
    else:  # slices of one projection; odd: from an address that is aligned to nothing but its type
        width = (hq + 2 * hk) * dim
        off = 1 if layout == "odd" else 0
        stride = width + (3 if layout == "odd" else 8 - width % 8)
        flat = dev(rn(g, n * stride + off), t)[off:].view(n, stride)[:, :width]
        q, k, v = (y.unflatten(1, (-1, dim)) for y in flat.split([hq * dim, hk * dim, hk * dim], 1))
    out = torch.full((n, hq, dim), 9.0, dtype=t, device="cuda")
    sl = 2.0 ** -np.arange(1, hq + 1, dtype=np.float32) if bias else None
    whole = before + after == 0
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, None if whole else i32(docs), None if prefix is None else i32(prefix), cap=cap,
                     slopes=None if sl is None else torch.from_numpy(sl).cuda())
    ctx.synchronize()
    ranges = plain.key_ranges(n, docs, prefix)
    want, size, top = plain.attention(host(q), host(k), host(v), ranges, dim ** -0.5, cap, sl)
    attention_close(host(out), want, size, top, EPS[ty])
    assert (host(out)[:before] == 0).all() and (host(out)[n - after:] == 0).all()


def test_attention_larger_scores_and_no_tokens(ctx):
    """Scores of hundreds (the running maximum moves far), and a row of no tokens."""
    g = gen(8)
    q, k, v = (dev(rn(g, 400, h, 64) * a, torch.bfloat16) for h, a in ((2, 20.0), (1, 8.0), (1, 1.0)))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out)
    ctx.synchronize()
    want, size, top = plain.attention(host(q), host(k), host(v), plain.key_ranges(400, None, None), 0.125)
    attention_close(host(out), want, size, top, EPS["bf16"])
    ocrhip.attention(ctx, q[:0], k[:0], v[:0], out[:0])
    no = i32([])
    ocrhip.attention(ctx, q, k, v, out, docs=i32([0]), prefix=no)
    ctx.synchronize()
    assert (host(out) == 0).all()


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 15])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_attention_of_documents_beside_bad_values(ctx, ty, dim, poison):
    """Keys and values that are not finite reach the queries that see them and no others."""
    g = gen(11)
    lens, n = [40, 30, 60], 130
    docs = np.concatenate([[0], np.cumsum(lens)])
    prefix = [0, 30, 10]
    q, k, v = (rn(g, n, h, dim) for h in (2, 1, 1))
    v[50:52, :, 1] = poison  # in the second document, which sees itself whole
    v[100] = poison  # late in the third, which is causal there
    k[125] = float("nan")
    q, k, v = (dev(x, TYPES[ty]) for x in (q, k, v))
    out = torch.zeros(n, 2, dim, dtype=TYPES[ty], device="cuda")
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, i32(docs), i32(prefix))
    ctx.synchronize()
    got = host(out)
    want, size, top = plain.attention(host(q), np.where(np.isnan(host(k)), 0, host(k)), np.where(np.isfinite(host(v)), host(v), 0),
                                      plain.key_ranges(n, docs, prefix), dim ** -0.5)
    clean = np.ones((n, 2, dim), bool)
    clean[40:70, :, 1] = False
    clean[100:] = False
    attention_close(got[clean], want[clean], size[clean], top, EPS[ty])
    for part in (got[40:70, :, 1], got[100:125]):
        assert (np.isnan(part) if np.isnan(poison) else part == poison).all()
    assert np.isnan(got[125:]).all()


DECODE = [
    # type, cache, heads, dim, page, cap, slopes
    ("f16", "f16", 8, 8, 64, 16, 0.0, False),
    ("bf16", "i8", 8, 2, 128, 16, 30.0, True),
    ("bf16", "e4m3", 16, 1, 128, 64, 0.0, True),
    ("f16", "i8", 3, 3, 80, 32, 0.0, False),
    ("f16", "e4m3", 6, 2, 96, 48, 10.0, False),
    ("bf16", "bf16", 24, 1, 128, 16, 0.0, True),
    ("f16", "i8", 2, 1, 256, 16, 0.0, False),
    ("bf16", "i8", 40, 1, 64, 16, 0.0, False),
    ("f16", "f16", 4, 2, 15, 7, 0.0, True),
    ("f16", "e4m3", 4, 4, 32, 16, 0.0, False),
    ("bf16", "bf16", 2, 2, 200, 33, 4.0, True),
]


def decode_case(g, fmt, hk, dim, page, lens, width=None):
    """A cache filled by hand at every sequence's positions: (cache memory, table, k, v), k and v
    [sequence][positions][heads][dim] float64; slots past a length hold junk."""
    table, pages, _ = tables(g, lens, page, width)
    mem = cache_memory(g, pages, hk, page, dim, fmt)
    kept = []
    for x in (0, 1):
        m, s = mem[x].cpu(), None if mem[2] is None else mem[2 + x].cpu()
        if fmt == "e4m3":  # NaN codes only as junk
            m = torch.where((m & 127) == 127, m ^ 1, m)
        if fmt in TYPES:
            m = torch.full(m.shape, float("nan")).to(TYPES[fmt])
        for r, n in enumerate(lens):
            for c in range(-(-n // page)):
                rows = min(page, n - c * page)
                p = table[r, c]
                if fmt in TYPES:
                    m[p, :, :rows] = rn(g, hk, rows, dim).to(TYPES[fmt])
                else:
                    s[p, :, :rows] = (0.5 + torch.rand(hk, rows, generator=g)) * (0.02 if fmt == "i8" else 0.008)
        mem[x] = m.cuda()
        if s is not None:
            mem[2 + x] = s.cuda()
        val = plain.e4m3_value(m.numpy()) if fmt == "e4m3" else m.double().numpy()
        if s is not None:
            val = val * s.double().numpy()[..., None]
        kept.append([np.concatenate([val[p].transpose(1, 0, 2) for p in table[r, : -(-n // page)]])[:n] if n else np.zeros((0, hk, dim))
                     for r, n in enumerate(lens)])
    return mem, table, kept[0], kept[1], pages


def decode_want(q, k, v, lens, scale, cap, sl):
    parts = [plain.attention(q[r:r + 1], k[r], v[r], ([0], [n]), scale, cap, sl, pos=[n - 1]) for r, n in enumerate(lens)]
    return np.concatenate([p[0] for p in parts]), np.concatenate([p[1] for p in parts]), max(p[2] for p in parts)


@pytest.mark.parametrize("ty,fmt,hq,hk,dim,page,cap,bias", DECODE)
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17, 33], [700, 3, 0, 255, 256, 257, 512], [5000, 31]])
def test_decode(ctx, ty, fmt, hq, hk, dim, page, cap, bias, lens):
    g = gen(sum(lens) + dim + page)
    mem, table, k, v, pages = decode_case(g, fmt, hk, dim, page, lens)
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    wide = dev(rn(g, len(lens), hq * dim + 8), TYPES[ty])
    q = wide[:, : hq * dim].unflatten(1, (hq, dim))
    out = torch.full((len(lens), hq, dim), 9.0, dtype=TYPES[ty], device="cuda")
    sl = 2.0 ** -np.arange(1, hq + 1, dtype=np.float32) if bias else None
    args = [i32(table), i32(lens), q, out]
    slopes = None if sl is None else torch.from_numpy(sl).cuda()
    torch.cuda.synchronize()
    cache.attend(*args, cap=cap, slopes=slopes)
    ctx.synchronize()
    want, size, top = decode_want(host(q), k, v, lens, dim ** -0.5, cap, sl)
    attention_close(host(out), want, size, top, EPS[ty], 3)
    for r, n in enumerate(lens):
        assert n or (host(out)[r] == 0).all()


def test_decode_shared_pages_and_holes(ctx):
    """Beams share their prompt's pages; a page that there is not counts as zeros."""
    g = gen(4)
    page, hk, hq, dim, n = 16, 2, 4, 64, 200
    mem, table, k, v, pages = decode_case(g, "i8", hk, dim, page, [n, n, n])
    table[1, :12] = table[0, :12]
    table[2, 3], table[2, 5] = -1, pages + 4
    k[1][:192], v[1][:192] = k[0][:192], v[0][:192]
    for c in (3, 5):
        k[2][c * page: c * page + page], v[2][c * page: c * page + page] = 0, 0
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, "i8", memory=mem)
    q = dev(rn(g, 3, hq, dim), torch.float16)
    out = torch.zeros_like(q)
    t, lens = i32(table), i32([n, n, n])
    torch.cuda.synchronize()
    cache.attend(t, lens, q, out)
    ctx.synchronize()
    want, size, top = decode_want(host(q), k, v, [n] * 3, dim ** -0.5, 0.0, None)
    attention_close(host(out), want, size, top, EPS["f16"], 3)


def test_prompt_and_single_token_agree(ctx):
    """The last token of a prompt by both forms: written by append, attended to in the cache."""
    g = gen(12)
    hq, hk, dim, n, page = 8, 2, 128, 333, 16
    qkv = dev(rn(g, n, (hq + 2 * hk) * dim), torch.bfloat16)
    table, pages, _ = tables(g, [n], page)
    mem = cache_memory(g, pages, hk, page, dim, "bf16")
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, "bf16", memory=mem)
    q, k = (torch.zeros(n, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, hk))
    out, last = torch.zeros_like(q), torch.zeros(1, hq, dim, dtype=torch.bfloat16, device="cuda")
    v = qkv[:, (hq + hk) * dim:].unflatten(1, (hk, dim))
    t, seq, pos, lens = i32(table), i32([0] * n), i32(range(n)), i32([n])
    torch.cuda.synchronize()
    cache.append(t, seq, pos, qkv, q, k)
    ocrhip.attention(ctx, q, k, v, out)
    cache.attend(t, lens, q[n - 1:], last)
    ctx.synchronize()
    want, size, top = plain.attention(host(q)[n - 1:], host(k), host(v), ([0], [n]), dim ** -0.5, pos=[n - 1])
    attention_close(host(out)[n - 1:], want, size, top, EPS["bf16"])
    attention_close(host(last), want, size, top, EPS["bf16"])


@pytest.mark.parametrize("fmt,dim,page", [("f16", 64, 16), ("i8", 128, 64), ("e4m3", 15, 7), ("bf16", 8, 1)])
@pytest.mark.parametrize("groups,beams", [(1, 1), (3, 4), (2, 32)])
def test_fork(ctx, fmt, dim, page, groups, beams):
    g = gen(beams + page)
    rows, hk = groups * beams, 2
    lens = [int(x) for x in torch.randint(0, 5 * page + 1, (rows,), generator=g)]
    if rows > 2:
        lens[1], lens[2] = 0, 2 * page
    table, pages, free = tables(g, lens, page, 6, rows)
    mem = cache_memory(g, pages, hk, page, dim, fmt, junk=False)
    if fmt in TYPES:
        mem[:2] = [dev(rn(g, *mem[0].shape), TYPES[fmt]) for _ in range(2)]
    else:
        mem[2:] = [torch.rand(mem[2].shape, generator=g).cuda() for _ in range(2)]
    parents = torch.randint(0, beams, (groups, beams), generator=g).numpy()
    if beams > 3:
        parents[0, 1], parents[0, 2] = -1, beams
    spare = np.asarray(free[:rows], np.int32)
    before = [None if m is None else m.cpu().clone() for m in mem]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    to, lo, us = (torch.full(s, 77, dtype=torch.int32, device="cuda") for s in (table.shape, (rows,), (rows,)))
    args = [i32(table), i32(lens), i32(parents), i32(spare)]
    torch.cuda.synchronize()
    cache.fork(*args, to, lo, us)
    ctx.synchronize()
    want = plain.fork(table, np.asarray(lens), parents, spare, page)
    for got, w in zip((to, lo, us), want):
        assert np.array_equal(host(got), w)
    for src, dst, n in want[3]:
        for b in before:
            if b is not None:
                b[dst, :, :n] = b[src, :, :n]
    for m, b in zip(mem, before):
        assert m is None or torch.equal(m.cpu().view(torch.uint8), b.view(torch.uint8))


def test_fork_of_bad_pages(ctx):
    """Pages that are not the pool's are neither read nor written; the tables still say what was asked."""
    page, hk, dim, pages = 4, 1, 8, 3
    mem = [torch.full((pages, hk, page, dim), 1.5, dtype=torch.float16, device="cuda") for _ in range(2)] + [None, None]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, "f16", memory=mem)
    table = np.array([[-1, 99], [2, 2]], np.int32)
    to, lo, us = i32(np.zeros((2, 2))), i32([0, 0]), i32([0, 0])
    for parents, lens, spare in (([[0, 0]], [6, 0], [1, 1]), ([[1, 1]], [0, 5], [-3, 500]), ([[1, 1]], [0, 3], [3, 2])):
        args = [i32(table), i32(lens), i32(parents), i32(spare)]
        torch.cuda.synchronize()
        cache.fork(*args, to, lo, us)
        ctx.synchronize()
        want = plain.fork(table, np.asarray(lens), np.asarray(parents), np.asarray(spare), page)
        assert np.array_equal(host(to), want[0]) and np.array_equal(host(us), want[2])
        assert (host(mem[0]) == 1.5).all() and (host(mem[1]) == 1.5).all()


def beam_check(ctx, logits, scores, finished, eos, in_place=False):
    g, w = scores.shape
    x = logits if isinstance(logits, torch.Tensor) else logits
    sc = torch.from_numpy(scores.astype(np.float32)).cuda()
    fin = None if finished is None else i32(finished)
    os, op, ot, of = torch.zeros(g, w, device="cuda"), i32(np.full((g, w), -5)), i32(np.full((g, w), -5)), i32(np.full((g, w), -5))
    if in_place:
        os, of = sc, fin
    want = plain.beam_select(host(x), scores.astype(np.float32), finished, -1 if eos is None else eos)
    torch.cuda.synchronize()
    ocrhip.beam_select(ctx, x, sc, fin, eos, os, op, ot, of)
    ctx.synchronize()
    assert np.array_equal(host(op), want[1]), (host(op), want[1])
    assert np.array_equal(host(ot), want[2]), (host(ot), want[2])
    if of is not None:
        assert np.array_equal(host(of), want[3])
    got = host(os)
    fine = np.isfinite(want[0])
    assert np.array_equal(got[~fine], want[0][~fine])
    # One rounding to float32, and the sum of the exponentials: 2^-21 of it.
    assert (np.abs(got[fine] - want[0][fine]) <= 2.0 ** -24 * np.abs(want[0][fine]) + 2.0 ** -21).all()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (2, 4, 97), (3, 5, 3), (2, 8, 18708), (1, 32, 50001), (5, 3, 8191), (1, 32, 2), (2, 2, 131072)])
def test_beam_select(ctx, ty, groups, beams, vocab):
    g = gen(vocab + beams)
    rows = groups * beams
    x = dev(rn(g, rows, vocab + 5) * 3, TYPES[ty])[:, :vocab]
    scores = -20 * torch.rand(groups, beams, generator=g).numpy()
    finished = (torch.rand(groups, beams, generator=g) < 0.3).int().numpy()
    beam_check(ctx, x, scores, finished, min(2, vocab - 1), in_place=True)
    beam_check(ctx, x, scores, None, None)
    scores[:, 1:] = -np.inf  # the first step
    beam_check(ctx, x, scores, None, 0)
    beam_check(ctx, x[:, :max(1, vocab - 3)], scores, np.zeros_like(finished), 0)


def test_beam_select_of_ties_and_holes(ctx):
    """Equal logits go to the lowest index; logits of minus infinity and NaN weigh nothing; plus
    infinity makes a row whose scores are no numbers."""
    v = 20000
    x = torch.zeros(8, v)
    x[1] = -float("inf")
    x[2, 5:] = -float("inf")
    x[3, ::2] = float("nan")
    x[4] = float("nan")
    x[5, 700] = float("inf")
    x[6] = torch.arange(v).float() % 3
    x[7] = -80 + torch.arange(v).float() % 2 * 160
    scores = np.array([[-1.0, -1.0], [-1.0, -1.0], [-1.0, -1.0], [-1.0, -1.0]])
    for t in (torch.float32, torch.bfloat16):
        beam_check(ctx, dev(x, t), scores, None, None)
        beam_check(ctx, dev(x, t), scores, np.array([[0, 1], [1, 0], [1, 1], [0, 0]]), v - 1)
        for w in (4, 8):
            beam_check(ctx, dev(x, t), np.full((8 // w, w), -2.5), None, 3)
    beam_check(ctx, dev(x[:2]), np.full((1, 2), -np.inf), None, 3)
    beam_check(ctx, dev(x[:2]), np.array([[-np.inf, np.nan]]), np.array([[1, 0]]), 3)


def test_other_streams(ctx):
    """Inputs made on a stream of torch's and outputs read there, ordered by acquire and release."""
    s = torch.cuda.Stream()
    g = gen(2)
    base = dev(rn(g, 2000, 4, 64))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        x = base
        for _ in range(50):
            x = x * 1.01 - 0.001 * x
        q = x.to(torch.float16)
        k, v = q[:, :2].contiguous(), q[:, 2:].contiguous()
        out = torch.zeros_like(q)
        ctx.acquire(s.cuda_stream)
        ocrhip.attention(ctx, q, k, v, out)
        ctx.release(s.cuda_stream)
        got = out * 1
    s.synchronize()
    ctx.synchronize()
    again = torch.zeros_like(q)
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, again)
    ctx.synchronize()
    assert torch.equal(got, again)


def test_arrays_of_the_library(ctx):
    """The same calls on the library's own device memory, without torch."""
    g = np.random.default_rng(1)
    n, hq, hk, dim = 50, 4, 2, 64
    host_arrays = [g.standard_normal((n, h, dim)).astype(np.float16) for h in (hq, hk, hk)]
    arrays = []
    for a in host_arrays:
        b = ctx.alloc(a.nbytes)
        b.upload(a)
        arrays.append(ocrhip.DeviceArray(b, a.shape, "f16"))
    out = ctx.alloc(n * hq * dim * 2)
    ocrhip.attention(ctx, *arrays, ocrhip.DeviceArray(out, (n, hq, dim), "f16"))
    got = out.download(np.float16, n * hq * dim).reshape(n, hq, dim).astype(np.float64)
    want, size, top = plain.attention(*host_arrays, plain.key_ranges(n, None, None), dim ** -0.5)
    attention_close(got, want, size, top, EPS["f16"])
    cache = ocrhip.KvCache(ctx, 3, 16, hk, dim, "e4m3")
    assert cache.k.shape == (3, hk, 16, dim)


def test_refusals_reach_the_caller(ctx):
    cache = ocrhip.KvCache(ctx, 3, 16, 2, 64, "f16")
    q = torch.zeros(1, 5, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ocrhip.OcrError, match="query heads"):
        cache.attend(i32([[0]]), i32([1]), q, torch.zeros_like(q))
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ocrhip.OcrError, match="16-bit cache"):
        cache.attend(i32([[0]]), i32([1]), q, torch.zeros_like(q))
    with pytest.raises(ocrhip.OcrError, match="overlap"):
        ocrhip.attention(ctx, q, q[:, :2].contiguous(), q[:, :2].contiguous(), q)
    with pytest.raises(ocrhip.OcrError, match="beams"):
        t = i32(np.zeros((40, 2)))
        o = i32(np.zeros(40))
        cache.fork(t, o, i32(np.zeros((1, 40))), o, i32(np.zeros((40, 2))), i32(np.zeros(40)), i32(np.zeros(40)))
