"""Latent attention on the GPU against float64 (oracle/text.py).

Weights are rounded once to the 16-bit type, half a step of the sum of p |v|, the output once more; scores are float32 sums,
off by 2^-21 of the largest, in the weight and its sum; exp is good to 2^-20."""
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


def close(got, want, size, top, eps):
    tol = (eps / 2 + 2.0 ** -18 + 2.0 ** -20 * top) * size + eps / 2 * np.abs(want) * (1 + eps) + 2.0 ** -24
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


def tables(g, lens, page, spare=2, width=None):
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g).tolist()
    t = np.full((len(lens), width or max(need + [1])), -1, np.int32)
    for r, c in enumerate(need):
        for e in range(c):
            t[r, e] = perm.pop()
    return t, pages


@pytest.mark.parametrize("tin,ty,rank,rot,pairs,normed,axes", [
    ("bf16", "bf16", 512, 64, "halves", True, None), ("f32", "f16", 128, 32, "adjacent", True, (8, 4, 4)),
    ("f16", "f16", 64, 64, "halves", False, (32,)), ("f32", "bf16", 37, 6, "adjacent", True, None),
    ("f16", "bf16", 200, 0, "halves", True, None), ("bf16", "f16", 1, 2, "halves", True, (0, 1)),
    ("f32", "f32", 0, 0, "", 0, 0), ("bf16", "bf16", 384, 128, "halves", True, (30, 34))])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_append(ctx, tin, ty, rank, rot, pairs, normed, axes, n):
    if rank == 0:
        with pytest.raises(ocrhip.OcrError, match="empty"):
            ocrhip.LatentCache(ctx, 1, 16, 0, 0)
        return
    g = gen(n + rank)
    page, width = 16, rank + rot
    table, pages = tables(g, [n], page)
    pool = torch.full((pages, page, width), 9.0, dtype=TYPES[ty], device="cuda")
    cache = ocrhip.LatentCache(ctx, pages, page, rank, rot, ty, memory=pool)
    x = rn(g, n, width + 3).to(TYPES[tin]).cuda()[:, :width]
    norm = (1 + 0.3 * rn(g, rank)).cuda() if normed else None
    order = torch.randperm(n, generator=g)
    pos, seq = i32(order), i32([0] * n)
    at = None if axes is None else torch.randint(0, 50000, (n, len(axes)), generator=g).to(torch.int32).cuda()
    out = torch.full((n, width), 9.0, dtype=TYPES[ty], device="cuda")
    t = i32(table)
    torch.cuda.synchronize()
    cache.append(t, seq, pos, x, out=out, norm=norm, eps=1e-5, theta=1e4, pairs=pairs, at=at, axes=axes, order="turns")
    ctx.synchronize()
    y = host(x)
    head = plain.norm(y[:, :rank], None if norm is None else host(norm), 1e-5)
    turn = plain.rotate_axes(y[:, None, rank:], host(pos)[:, None] if at is None else host(at), 0, rot, 1e4, pairs, axes or (rot // 2,),
                             "turns", "shared")[:, 0]
    want, got = np.concatenate([head, turn], 1), host(out)
    top = np.concatenate([np.abs(p) * 0 + np.abs(p).max(1, keepdims=True, initial=0) for p in (head, turn)], 1)
    assert (np.abs(got - want) <= EPS[ty] / 2 * np.abs(want) + 2.0 ** -20 * top + 2.0 ** -24).all()
    held = host(pool)
    for i, p in enumerate(order.tolist()):
        assert np.array_equal(held[table[0, p // page], p % page], got[i])
    assert (held == 9).all(-1).sum() >= pages * page - n  # nothing else is written


def test_append_drops_what_has_no_place(ctx):
    pool = torch.full((3, 16, 48), 9.0, dtype=torch.float16, device="cuda")
    cache = ocrhip.LatentCache(ctx, 3, 16, 32, 16, "f16", memory=pool)
    x = torch.ones(6, 48, device="cuda")
    t, seq, pos = i32([[2, -1], [7, 0]]), i32([0, 0, -1, 2, 1, 1]), i32([3, 17, 0, 0, 2, 32])
    torch.cuda.synchronize()
    cache.append(t, seq, pos, x)
    cache.append(t[:0], seq[:0], pos[:0], x[:0])
    ctx.synchronize()
    changed = (host(pool) != 9).any(-1)
    assert changed.sum() == 1 and changed[2, 3]


ATTEND = [
    # type, heads, rank, rot, page
    ("bf16", 128, 512, 64, 64), ("f16", 16, 512, 64, 16), ("bf16", 5, 384, 32, 16), ("f16", 40, 128, 32, 32), ("bf16", 1, 256, 64, 7),
    ("f16", 17, 64, 64, 16), ("bf16", 3, 37, 6, 16), ("f16", 2, 512, 128, 16), ("bf16", 33, 32, 0, 16), ("f16", 64, 448, 8, 1),
    ("f16", 9, 8, 8, 16), ("bf16", 130, 96, 32, 16),
]


def attend_case(ctx, g, ty, heads, rank, rot, page, lens, pad=0, width=None):
    w = rank + rot
    table, pages = tables(g, lens, page, width=width)
    pool = torch.full((pages, page, w), float("nan"), dtype=TYPES[ty])  # junk in the slots past every length
    for r, n in enumerate(lens):
        for p in range(0, n, page):
            pool[table[r, p // page], : min(page, n - p)] = rn(g, min(page, n - p), w).to(TYPES[ty])
    cache = ocrhip.LatentCache(ctx, pages, page, rank, rot, ty, memory=pool.cuda())
    q = rn(g, len(lens), heads * w + pad).to(TYPES[ty]).cuda()[:, : heads * w].unflatten(1, (heads, w))
    out = torch.full((len(lens), heads * rank + pad), 9.0, dtype=TYPES[ty], device="cuda")
    t, ls = i32(table), i32(lens)
    torch.cuda.synchronize()
    cache.attend(t, ls, q, out[:, : heads * rank].unflatten(1, (heads, rank)), scale=w ** -0.5)
    ctx.synchronize()
    got, held, qs = host(out), pool.double().numpy(), host(q)
    for r, n in enumerate(lens):
        c = np.concatenate([held[table[r, e]] for e in range(-(-n // page))])[:n] if n else np.zeros((0, w))
        want, size, top = plain.latent(qs[r], c, rank, w ** -0.5)
        close(got[r, : heads * rank].reshape(heads, rank), want, size, top, EPS[ty])
    assert (got[:, heads * rank:] == 9).all()


@pytest.mark.parametrize("ty,heads,rank,rot,page", ATTEND)
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17, 33, 64], [700, 3, 0, 255, 256, 257], [4100, 31]])
def test_attend(ctx, ty, heads, rank, rot, page, lens):
    attend_case(ctx, gen(sum(lens) + rank), ty, heads, rank, rot, page, lens)


@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("heads", [16, 128])
def test_attend_rows_apart(ctx, heads, pad):
    attend_case(ctx, gen(pad), "bf16", heads, 128, 64, 16, [70, 5], pad)


def test_attend_wide_tables_and_holes(ctx):
    """A table far wider than the lengths, pages that there are not (zeros), lengths past the table."""
    g = gen(4)
    attend_case(ctx, g, "bf16", 16, 128, 64, 16, [300, 20], width=5000)
    for rank, rot, heads in ((128, 64, 20), (20, 4, 3)):
        w, page, n = rank + rot, 16, 200
        table, pages = tables(g, [n, n], page)
        pool = rn(g, pages, page, w).to(torch.float16)
        c = [pool.double().numpy()[table[r]].reshape(-1, w)[:n].copy() for r in range(2)]
        table[0, 2], table[0, 12], table[1, 0] = -1, pages + 3, -9
        c[0][32:48], c[0][192:], c[1][:16] = 0, 0, 0
        pool[0] = torch.where(torch.isin(torch.tensor(0), torch.from_numpy(table)), pool[0], float("nan"))
        cache = ocrhip.LatentCache(ctx, pages, page, rank, rot, "f16", memory=pool.cuda())
        q = rn(g, 2, heads, w).to(torch.float16).cuda()
        out = torch.zeros(2, heads, rank, dtype=torch.float16, device="cuda")
        t, ls = i32(table), i32([n, 2000000000])
        torch.cuda.synchronize()
        cache.attend(t, ls, q, out, scale=0.1)
        ctx.synchronize()
        c[1] = np.concatenate([np.zeros((16, w)), pool.double().numpy()[table[1, 1:]].reshape(-1, w)])
        for r in range(2):
            want, size, top = plain.latent(host(q)[r], c[r], rank, 0.1)
            close(host(out)[r], want, size, top, EPS["f16"])


def test_attend_large_scores(ctx):
    g = gen(14)
    pool = (rn(g, 30, 16, 192) * 8).to(torch.bfloat16).cuda()
    cache = ocrhip.LatentCache(ctx, 30, 16, 128, 64, "bf16", memory=pool)
    q = (rn(g, 1, 16, 192) * 6).to(torch.bfloat16).cuda()
    out = torch.empty(1, 16, 128, dtype=torch.bfloat16, device="cuda")
    t = i32([range(30)])
    torch.cuda.synchronize()
    for scale in (0.3, -0.3, 0.0):
        cache.attend(t, i32([471]), q, out, scale=scale)
        ctx.synchronize()
        want, size, top = plain.latent(host(q)[0], host(pool).reshape(-1, 192)[:471], 128, scale)
        close(host(out)[0], want, size, top, EPS["bf16"])


@pytest.mark.parametrize("ty,rank,rot,page", [("bf16", 512, 64, 16), ("f16", 37, 6, 7)])
def test_fork(ctx, ty, rank, rot, page):
    g = gen(rank)
    lens = [20, 20, 33, 5, page, 0]
    table, pages = tables(g, lens, page, spare=8)
    spare = np.setdiff1d(np.arange(pages), table)[:6].astype(np.int32)
    pool = rn(g, pages, page, rank + rot).to(TYPES[ty]).cuda()
    want_pool = pool.cpu().clone()
    cache = ocrhip.LatentCache(ctx, pages, page, rank, rot, ty, memory=pool)
    parents = np.array([[1, 1, 0], [0, 0, 7]], np.int32)
    out = [torch.full(s, -9, dtype=torch.int32, device="cuda") for s in (table.shape, (6,), (6,))]
    args = [i32(table), i32(lens), i32(parents), i32(spare)]
    torch.cuda.synchronize()
    cache.fork(*args, *out)
    ctx.synchronize()
    t, n, used, copies = plain.fork(table, np.asarray(lens), parents, spare, page)
    for got, want in zip(out, (t, n, used)):
        assert np.array_equal(host(got), want)
    for a, b, tail in copies:
        want_pool[b, :tail] = want_pool[a, :tail]
    assert torch.equal(pool.cpu(), want_pool)


PROMPTS = [
    # type, heads, key, rot, value, documents, prefix
    ("bf16", 4, 128, 64, 128, [300], None), ("f16", 3, 64, 32, 64, [17, 1, 0, 64, 129], [3, 1, 0, 64, 500]), ("f16", 2, 96, 32, 64, [150, 40], None),
    ("bf16", 1, 32, 64, 128, [513], [512]), ("f16", 2, 128, 0, 128, [90], [20]), ("bf16", 2, 15, 6, 21, [70, 20], [0, 20]),
    ("f16", 1, 256, 128, 256, [40], None), ("bf16", 2, 40, 8, 72, [200], [10]), ("bf16", 20, 128, 64, 128, [700, 1, 500], [650, 0, 0]),
    ("f16", 1, 1, 2, 1, [66], None), ("bf16", 1, 128, 64, 64, [1100], [100]),
]


@pytest.mark.parametrize("ty,heads,key,rot,value,lens,prefix", PROMPTS)
@pytest.mark.parametrize("layout", ["apart", "beside", "odd"])
def test_prompts(ctx, ty, heads, key, rot, value, lens, prefix, layout):
    g = gen(sum(lens) + key + rot)
    before, after = (0, 0) if len(lens) == 1 and layout == "apart" else (5, 9)
    n = sum(lens) + before + after
    docs = before + np.concatenate([[0], np.cumsum(lens)])
    t = TYPES[ty]
    cut = lambda *shape: rn(g, *shape).to(t).cuda()  # noqa: E731
    q = cut(n, heads, key + rot)
    if layout == "apart":
        k, v, r = cut(n, heads, key), cut(n, heads, value), cut(n, rot)
    else:
        off = 1 if layout == "odd" else 0
        up = cut(n * heads * (key + value + off) + off)[off:].view(n, heads, key + value + off)
        k, v, r = up[..., :key], up[..., key: key + value], cut(n, 24 + rot + off)[:, 24 + off:]
    out = torch.full((n, heads, value), 9.0, dtype=t, device="cuda")
    whole = before + after == 0
    scale = (key + rot) ** -0.5
    torch.cuda.synchronize()
    ocrhip.latent_attention(ctx, q, k, r if rot else None, v, out, None if whole else i32(docs), None if prefix is None else i32(prefix))
    ctx.synchronize()
    want, size, top = plain.latent_prompt(host(q), host(k), host(r) if rot else None, host(v), plain.key_ranges(n, docs, prefix), scale)
    close(host(out), want, size, top, EPS[ty])
    assert (host(out)[:before] == 0).all() and (host(out)[n - after:] == 0).all()


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("key,rot,value", [(128, 64, 128), (15, 6, 21)])
def test_prompts_beside_bad_values(ctx, key, rot, value, poison):
    """Values that are not finite reach the queries that see them and no others."""
    g = gen(11)
    lens, n = [40, 30, 60], 130
    docs, prefix = np.concatenate([[0], np.cumsum(lens)]), [0, 30, 10]
    q, k, r, v = rn(g, n, 2, key + rot), rn(g, n, 2, key), rn(g, n, rot), rn(g, n, 2, value)
    v[50:52, :, 1] = poison
    v[100] = poison
    r[125] = float("nan")
    q, k, r, v = (x.to(torch.bfloat16).cuda() for x in (q, k, r, v))
    out = torch.zeros(n, 2, value, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ocrhip.latent_attention(ctx, q, k, r, v, out, i32(docs), i32(prefix))
    ctx.synchronize()
    got = host(out)
    want, size, top = plain.latent_prompt(host(q), host(k), np.nan_to_num(host(r)), np.where(np.isfinite(host(v)), host(v), 0),
                                          plain.key_ranges(n, docs, prefix), (key + rot) ** -0.5)
    clean = np.ones(got.shape, bool)
    clean[40:70, :, 1] = False
    clean[100:] = False
    close(got[clean], want[clean], size[clean], top, EPS["bf16"])
    for part in (got[40:70, :, 1], got[100:125]):
        assert (np.isnan(part) if np.isnan(poison) else part == poison).all()
    assert np.isnan(got[125:]).all()


def test_absorbed_and_expanded_agree(ctx):
    """A prompt's last token by both forms, with the same expansions: cache, rotation and both attentions together."""
    g = gen(30)
    n, heads, key, rot, value, rank, page = 200, 4, 64, 32, 64, 128, 16
    x = rn(g, n, rank + rot).to(torch.bfloat16).cuda()
    up_k, up_v = (rn(g, heads, rank, d).mul(rank ** -0.5).to(torch.bfloat16).cuda() for d in (key, value))
    q = rn(g, n, heads, key + rot).to(torch.bfloat16).cuda()
    pos = i32(range(n))
    cache = ocrhip.LatentCache(ctx, 16, page, rank, rot, "bf16")
    table, seq, lens = i32([range(16)]), i32([0] * n), i32([n])
    c = torch.empty(n, rank + rot, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    cache.append(table, seq, pos, x, out=c)
    ocrhip.rotate(ctx, q, pos, first=key, rot=rot)
    ctx.synchronize()
    lat = c[:, :rank].float()
    k, v = (torch.stack([lat @ u[h].float() for h in range(heads)], 1).to(torch.bfloat16) for u in (up_k, up_v))
    out = torch.empty(n, heads, value, dtype=torch.bfloat16, device="cuda")
    absorbed = torch.cat([torch.stack([q[-1:, h, :key].float() @ up_k[h].float().T.contiguous() for h in range(heads)], 1).to(torch.bfloat16),
                          q[-1:, :, key:]], 2)
    last = torch.empty(1, heads, rank, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    scale = (key + rot) ** -0.5
    ocrhip.latent_attention(ctx, q, k, c[:, rank:], v, out, scale=scale)
    cache.attend(table, lens, absorbed, last, scale=scale)
    ctx.synchronize()
    ends = torch.stack([last[0, h].float() @ up_v[h].float() for h in range(heads)])
    # Each form rounds keys or queries, weights and sums to bfloat16: five half steps, of values up to a few.
    size = host(v).__abs__().max()
    assert np.abs(host(ends) - host(out)[-1]).max() <= 5 * 2.0 ** -8 * size
