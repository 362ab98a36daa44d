"""Attention weights added up, and eviction by them, on the GPU against float64 (oracle/text.py).

A weight is e^(s - m) / sum: scores are float32 sums, off by 2^-21 of the largest, in the weight and in its sum; exp and
tanh are good to 2^-20; sums of N weights, over at least 16 lanes, lose N / 16 + 16 times 2^-24 of themselves."""
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


def weights_close(got, want, before, top, terms):
    tol = (2.0 ** -18 + 2.0 ** -20 * top + (terms / 16 + 16) * 2.0 ** -24) * want + 2.0 ** -23 * (want + np.abs(before)) + 2.0 ** -28
    bad = np.abs(got - (before + want)) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], (before + want)[bad][:5])


PROMPTS = [
    # type, heads, dim, documents, prefix, cap, slopes, window
    ("f16", 2, 2, 64, [1], None, 0.0, False, None),
    ("bf16", 4, 1, 64, [109], [109], 0.0, False, None),
    ("bf16", 4, 2, 128, [17, 1, 0, 64, 129], [3, 1, 0, 64, 500], 0.0, True, 10),
    ("f16", 2, 1, 128, [300], [77], 20.0, False, None),
    ("f16", 3, 3, 32, [31, 33, 200], None, 0.0, True, 1),
    ("bf16", 8, 1, 80, [513], [512], 50.0, True, None),
    ("f16", 6, 2, 96, [63, 65, 127], [10, 0, 127], 5.0, True, 64),
    ("bf16", 2, 2, 256, [150], [40], 0.0, False, 33),
    ("f16", 2, 1, 15, [140], [20], 0.0, True, None),
    ("bf16", 1, 1, 128, [1100], [100], 0.0, False, None),
    ("f16", 16, 2, 64, [700, 1, 500], [650, 0, 0], 0.0, False, 500),
    ("bf16", 2, 1, 72, [200, 5], [0, 5], 1e6, False, 1000),
]


@pytest.mark.parametrize("ty,hq,hk,dim,lens,prefix,cap,bias,window", PROMPTS)
@pytest.mark.parametrize("layout", ["apart", "odd"])
def test_prompt_weights(ctx, ty, hq, hk, dim, lens, prefix, cap, bias, window, layout):
    g = gen(sum(lens) + dim)
    before, after = (0, 0) if len(lens) == 1 and layout == "apart" else (5, 9)
    n = sum(lens) + before + after
    docs = before + np.concatenate([[0], np.cumsum(lens)])
    t = TYPES[ty]
    off = 1 if layout == "odd" else 0
    width = (hq + 2 * hk) * dim + 3 * off
    flat = rn(g, n * width + off).to(t).cuda()[off:].view(n, width)[:, : (hq + 2 * hk) * dim]
    q, k, v = (y.unflatten(1, (-1, dim)) for y in flat.split([hq * dim, hk * dim, hk * dim], 1))
    out, same = (torch.full((n, hq, dim), 9.0, dtype=t, device="cuda") for _ in range(2))
    sl = 2.0 ** -np.arange(1, hq + 1, dtype=np.float32) if bias else None
    slopes = None if sl is None else torch.from_numpy(sl).cuda()
    whole = before + after == 0
    ds, ps = None if whole else i32(docs), None if prefix is None else i32(prefix)
    most = max(lens) + 3
    start = torch.rand(len(lens), hk, most, generator=g)
    w = start.clone().cuda()
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, ds, ps, cap=cap, slopes=slopes, weights=w, window=window)
    ocrhip.attention(ctx, q, k, v, same, ds, ps, cap=cap, slopes=slopes)
    ctx.synchronize()
    assert torch.equal(out, same)  # the outputs do not depend on the weights
    want, top = plain.prompt_weights(host(q), host(k), docs, prefix, dim ** -0.5, cap, sl, window)
    weights_close(host(w)[..., : max(lens)], want, start.double().numpy()[..., : max(lens)], top, max(lens) * hq // hk)
    for d, c in enumerate(lens):  # places of no key stay
        assert torch.equal(w.cpu()[d, :, c:], start[d, :, c:])


def test_prompt_weights_of_few_places_and_junk(ctx):
    """Places past the array are dropped, and documents beside values that are not finite keep their weights."""
    g = gen(2)
    lens, n = [70, 40, 90], 200
    docs = np.concatenate([[0], np.cumsum(lens)])
    q, k, v = (rn(g, n, h, 64) for h in (4, 2, 2))
    k[80] = float("nan")
    k[90] = float("inf")
    v[120:] = float("nan")
    q, k, v = (x.to(torch.bfloat16).cuda() for x in (q, k, v))
    guard = torch.full((3 * 2 * 50 + 64,), 7.0, device="cuda")
    w = guard[:300].view(3, 2, 50)
    w.zero_()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, k, v, out, i32(docs), weights=w)
    ctx.synchronize()
    want, top = plain.prompt_weights(host(q), np.nan_to_num(host(k)), docs, None, 0.125)
    got = host(w)
    for d in (0, 2):
        weights_close(got[d], want[d][..., :50], np.zeros_like(got[d]), top, 180)
    assert (host(guard)[300:] == 7).all()
    assert np.isnan(got[1][:, :40]).all()  # all of its keys are seen by a query with such a score


def test_prompt_weights_of_no_documents(ctx):
    q = rn(gen(1), 9, 2, 64).to(torch.float16).cuda()
    out = torch.full_like(q, 3.0)
    torch.cuda.synchronize()
    ocrhip.attention(ctx, q, q, q, out, docs=i32([0]), weights=torch.zeros(0, 2, 9, device="cuda"))
    ocrhip.attention(ctx, q, q, q, out, weights=torch.zeros(1, 2, 0, device="cuda"))
    ctx.synchronize()
    assert np.isfinite(host(out)).all() and (host(out) != 3).all()


def paged(g, fmt, hk, dim, page, lens, width=None):
    """A cache filled by hand, junk past every length: (memory, table, keys, values), those a float64 [positions][heads][dim] a sequence."""
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 2, width or max(need + [1])
    perm = torch.randperm(pages, generator=g).tolist()
    table = np.full((len(lens), width), -1, np.int32)
    for r, c in enumerate(need):
        for e in range(c):
            table[r, e] = perm.pop()
    shape = (pages, hk, page, dim)
    mem, kept = [], []
    for _ in range(2):
        if fmt == "i8":
            m = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
        elif fmt == "e4m3":
            m = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
            m = torch.where((m & 127) == 127, m ^ 1, m)
        else:
            m = rn(g, *shape).to(TYPES[fmt])
        s = (0.5 + torch.rand(shape[:3], generator=g)) * (0.02 if fmt == "i8" else 0.008) if fmt in plain.QMAX else None
        junk = torch.ones(shape[:3], dtype=torch.bool)
        for r, n in enumerate(lens):
            for e in range(need[r]):
                junk[table[r, e], :, : min(page, n - e * page)] = False
        if s is None:
            m[junk] = float("nan")
        else:
            s[junk] = float("nan")
        val = plain.e4m3_value(m.numpy()) if fmt == "e4m3" else m.double().numpy()
        val = val if s is None else val * s.double().numpy()[..., None]
        kept.append([np.concatenate([val[p].transpose(1, 0, 2) for p in table[r, : need[r]]])[:n] if n else np.zeros((0, hk, dim))
                     for r, n in enumerate(lens)])
        mem.append((m.cuda(), None if s is None else s.cuda()))
    return [mem[0][0], mem[1][0], mem[0][1], mem[1][1]], table, kept[0], kept[1], pages


SINGLE = [
    ("f16", "f16", 8, 8, 64, 16, 0.0, False),
    ("bf16", "i8", 8, 2, 128, 16, 30.0, True),
    ("bf16", "e4m3", 16, 1, 128, 64, 0.0, True),
    ("f16", "i8", 3, 3, 80, 32, 0.0, False),
    ("bf16", "bf16", 24, 1, 128, 16, 0.0, True),
    ("f16", "i8", 2, 1, 256, 16, 0.0, False),
    ("bf16", "i8", 40, 1, 64, 16, 0.0, False),
    ("f16", "f16", 4, 2, 15, 7, 0.0, True),
    ("bf16", "bf16", 2, 2, 200, 33, 4.0, True),
]


@pytest.mark.parametrize("ty,fmt,hq,hk,dim,page,cap,bias", SINGLE)
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17, 33], [700, 3, 0, 255, 256, 257, 512], [5000, 31]])
def test_single_weights(ctx, ty, fmt, hq, hk, dim, page, cap, bias, lens):
    g = gen(sum(lens) + dim + page)
    mem, table, k, v, pages = paged(g, fmt, hk, dim, page, lens)
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    q = rn(g, len(lens), hq, dim).to(TYPES[ty]).cuda()
    out, same = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    sl = 2.0 ** -np.arange(1, hq + 1, dtype=np.float32) if bias else None
    slopes = None if sl is None else torch.from_numpy(sl).cuda()
    most = max(lens) + 5 if lens[0] != 700 else 501  # some places past the array
    start = torch.rand(len(lens), hk, most, generator=g)
    w, t, ls = start.clone().cuda(), i32(table), i32(lens)
    torch.cuda.synchronize()
    cache.attend(t, ls, q, out, cap=cap, slopes=slopes, weights=w)
    cache.attend(t, ls, q, same, cap=cap, slopes=slopes)
    ctx.synchronize()
    assert torch.equal(out, same)
    qs, before = host(q), start.double().numpy()
    want, top = np.zeros(start.shape), 0.0
    for r, n in enumerate(lens):
        for h in range(hq if n else 0):
            s = k[r][:, h // (hq // hk)] @ qs[r, h] * dim ** -0.5
            bias_ = 0.0 if sl is None else -float(sl[h]) * np.arange(n - 1, -1, -1)
            want[r, h // (hq // hk), :n] += plain.weights(s, cap, bias_)[:most]
            top = max(top, np.abs(s).max())
    weights_close(host(w), want, before, top, hq // hk)
    for r, n in enumerate(lens):
        assert torch.equal(w.cpu()[r, :, n:], start[r, :, n:])


def evict_case(ctx, g, fmt, hk, dim, page, lens, most, weights, held, newest, keep, first, recent, in_place, table=None, mem=None):
    """The call, checked against the oracle vector by vector; (memory, table) afterwards."""
    if mem is None:
        mem, table, _, _, pages = paged(g, fmt, hk, dim, page, lens)
    pages = mem[0].shape[0]
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, fmt, memory=mem)
    old = [None if m is None else m.cpu().clone() for m in mem]
    w, h, t, ls, ns = torch.from_numpy(weights).cuda(), i32(held), i32(table), i32(lens), i32(newest)
    wo, ho = (w, h) if in_place else (torch.full_like(w, 5.0), torch.full_like(h, 5))
    lo = i32([-7] * len(lens))
    torch.cuda.synchronize()
    cache.evict(t, ls, ns, w, h, keep, lo, first=first, recent=recent, **({} if in_place else {"weights_out": wo, "held_out": ho}))
    ctx.synchronize()
    got_w, got_h, got_l = wo.cpu().numpy(), ho.cpu().numpy(), lo.cpu().numpy()
    for r, n in enumerate(lens):
        n = max(0, min(n, table.shape[1] * page, most))
        assert got_l[r] == min(n, keep)
        for x in range(hk):
            moves, ww, hh = plain.evict(weights[r, x], held[r, x], n, newest[r], keep, first, recent)
            assert np.array_equal(got_w[r, x], ww, equal_nan=True), (r, x)
            assert np.array_equal(got_h[r, x], hh), (r, x)
            for a, b in moves:
                src, dst = table[r, a // page], table[r, b // page]
                if not (0 <= src < pages and 0 <= dst < pages):
                    continue
                for m in old:
                    if m is not None:
                        m[dst, x, b % page] = m[src, x, a % page]
    for m, want in zip(mem, old):
        assert m is None or np.array_equal(m.cpu().view(torch.uint8).numpy(), want.view(torch.uint8).numpy())  # all of the pool, bit by bit
    return mem, table


EVICT = [
    # cache, heads, dim, page, lengths, places more than needed, keep, first, recent
    ("f16", 4, 64, 16, [100, 40, 41, 0, 1, 99], 0, 40, 4, 8),
    ("bf16", 2, 128, 64, [1000, 700, 301], 7, 300, 0, 0),
    ("i8", 3, 80, 7, [50, 33, 1], 3, 32, 2, 30),
    ("e4m3", 1, 15, 33, [200, 150], 0, 1, 0, 1),
    ("f16", 1, 64, 16, [5000, 4097, 64], 0, 4096, 4, 64),
    ("bf16", 1, 32, 16, [70000, 300], 0, 2000, 1, 500),
    ("f16", 2, 1, 1, [9, 8, 7], 2, 8, 8, 0),
    ("bf16", 1, 64, 16, [33000, 32000], 0, 31999, 4, 100),
]


@pytest.mark.parametrize("fmt,hk,dim,page,lens,more,keep,first,recent", EVICT)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(ctx, fmt, hk, dim, page, lens, more, keep, first, recent, kind):
    if kind != "spread" and max(lens) > 40000:
        lens = [6000, 300]
    g = gen(sum(lens) + keep)
    most = max(lens) + more
    shape = (len(lens), hk, most)
    w = torch.rand(shape, generator=g).pow(4)
    if kind == "ties":  # few different weights, most of them zero
        w = torch.randint(0, 3, shape, generator=g).clamp(min=1).sub(1).float() * 0.25
    held = torch.full(shape, -1, dtype=torch.int32)
    if kind == "odd":
        w[torch.rand(shape, generator=g) < 0.1] = float("nan")
        w[torch.rand(shape, generator=g) < 0.05] = -0.0
        w[torch.rand(shape, generator=g) < 0.05] = float("inf")
        w[torch.rand(shape, generator=g) < 0.05] = -float("inf")
        held = torch.where(torch.rand(shape, generator=g) < 0.5, torch.randint(0, 2 * most, shape, generator=g), -1).to(torch.int32)
    newest = [n + 10 * r for r, n in enumerate(lens)]
    evict_case(ctx, g, fmt, hk, dim, page, lens, most, w.numpy(), held.numpy(), newest, keep, first, recent, kind == "ties")


def test_evict_step_by_step(ctx):
    """Tokens come one at a time and the cache stays at its size: what is held are the tokens that should be."""
    g = gen(9)
    hk, dim, page, keep, first, recent = 2, 32, 8, 24, 2, 6
    lens, most = [25], 25
    mem, table, k, _, pages = paged(g, "f16", hk, dim, page, lens, width=4)
    w, held = torch.rand(1, hk, most, generator=g).numpy(), np.full((1, hk, most), -1, np.int32)
    mine = [{p: float(w[0, x, p]) for p in range(25)} for x in range(hk)]  # position: weight
    for newest in range(24, 60):
        evict_case(ctx, g, "f16", hk, dim, page, lens, most, w, held, [newest], keep, first, recent, False, table, mem)
        nw, nh = np.zeros_like(w), np.full_like(held, -1)
        for x in range(hk):
            _, nw[0, x], nh[0, x] = plain.evict(w[0, x], held[0, x], 25, newest, keep, first, recent)
            drop = min((p for p in mine[x] if first <= p <= newest - recent), key=lambda p: mine[x][p])
            del mine[x][drop]
            assert sorted(nh[0, x, :keep]) == sorted(mine[x])
            nw[0, x] += np.where(nh[0, x] >= 0, torch.rand(most, generator=g).numpy(), 0).astype(np.float32)
            for p, y in zip(nh[0, x, :keep], nw[0, x, :keep]):
                mine[x][int(p)] = float(y)
            mine[x][newest + 1] = 0.0
        w, held = nw, nh


def test_evict_of_bad_pages_and_lengths(ctx):
    """Pages that there are not are neither read nor written; lengths past the table or the arrays are cut."""
    g = gen(6)
    hk, dim, page, most = 2, 64, 16, 90
    lens = [90, 2000000000, -3]
    mem, table, _, _, pages = paged(g, "f16", hk, dim, page, [96, 96, 96])
    table[0, 4], table[0, 1], table[1, 5], table[1, 0] = -1, pages + 7, pages, -2
    w = torch.rand(3, hk, most, generator=g).numpy()
    evict_case(ctx, g, "f16", hk, dim, page, lens, most, w, np.full((3, hk, most), -1, np.int32), [89, 89, 5], 50, 2, 4, False, table, mem)


def test_evict_positions_at_the_end_of_the_numbers(ctx):
    """The newest position near 2^31, and positions held at it."""
    g = gen(7)
    w = torch.rand(1, 1, 40, generator=g).numpy()
    held = np.where(np.arange(40) % 3 == 0, 2 ** 31 - 1 - np.arange(40), -1).astype(np.int32)[None, None]
    evict_case(ctx, g, "f16", 1, 64, 16, [40], 40, w, held, [2 ** 31 - 1], 20, 0, 20, False)


def test_a_bounded_cache_as_it_is_used(ctx):
    """Prompt, weights, eviction, then tokens written after it: attention over what is left is that over the kept tokens."""
    g = gen(21)
    hq, hk, dim, page, n, keep = 8, 2, 64, 16, 150, 64
    qkv = rn(g, n + 1, (hq + 2 * hk) * dim).to(torch.bfloat16).cuda()
    cache = ocrhip.KvCache(ctx, 12, page, hk, dim, "bf16")
    table, seq = i32([range(12)]), i32([0] * n)
    q, k = (torch.empty(n, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, hk))
    v = qkv[:n, (hq + hk) * dim:].unflatten(1, (hk, dim))
    out = torch.empty_like(q)
    w, held = torch.zeros(1, hk, n + 1, device="cuda"), torch.full((1, hk, n + 1), -1, dtype=torch.int32, device="cuda")
    lens = i32([0])
    args = [i32(range(n)), i32([n]), i32([n - 1]), i32([0]), i32([keep]), i32([n])]
    torch.cuda.synchronize()
    cache.append(table, seq, args[0], qkv[:n], q, k)
    ocrhip.attention(ctx, q, k, v, out, weights=w)
    ctx.synchronize()
    before = w.clone()
    torch.cuda.synchronize()
    cache.evict(table, args[1], args[2], w, held, keep, lens, first=4, recent=16)
    one, ko = (torch.empty(1, h, dim, dtype=torch.bfloat16, device="cuda") for h in (hq, hk))
    cache.append(table, args[3], args[4], qkv[n:], one, ko, at=args[5])  # the next place, turned by its position
    last, after = torch.empty_like(one), i32([keep + 1])
    ctx.synchronize()
    w2 = w.clone()
    torch.cuda.synchronize()
    cache.attend(table, after, one, last, weights=w)
    ctx.synchronize()
    assert host(lens)[0] == keep
    ks, vs = np.concatenate([host(k), host(ko)]), host(qkv[:, (hq + hk) * dim:].unflatten(1, (hk, dim)))
    gain = host(w) - host(w2)
    for x in range(hk):
        there = host(held)[0, x, :keep]
        _, ww, hh = plain.evict(before.cpu().numpy()[0, x], np.full(n + 1, -1, np.int32), n, n - 1, keep, 4, 16)
        assert np.array_equal(hh[:keep], there) and {0, 1, 2, 3, *range(n - 16, n)} <= set(there.tolist())
        at = np.concatenate([there, [n]])
        for h in range(x * hq // hk, (x + 1) * hq // hk):
            p = plain.weights(ks[at, x] @ host(one)[0, h] * dim ** -0.5, 0.0, 0.0)
            want, size = p @ vs[at, x], p @ np.abs(vs[at, x])
            assert (np.abs(host(last)[0, h] - want) <= (3 * 2.0 ** -8 + 2.0 ** -14) * size + 2.0 ** -8 * np.abs(want)).all()
        total = sum(plain.weights(ks[at, x] @ host(one)[0, h] * dim ** -0.5, 0.0, 0.0) for h in range(x * hq // hk, (x + 1) * hq // hk))
        assert (np.abs(gain[0, x, : keep + 1] - total) <= 2.0 ** -16 * total + 2.0 ** -20).all()
