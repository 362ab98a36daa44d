"""The text decoder's further operators as programs call them: which kernel each call runs, the same results twice, without the
native module, on another stream and on the library's own memory, many sequences, pools past 32 bits, refusals."""
import numpy as np
import pytest
import torch

import ocrhip
from ocrhip import text
from oracle import text as plain
from test_gpu_text_forms import FORMS
from test_gpu_text_latent import EPS, close, gen, host, i32, rn, tables

pytestmark = pytest.mark.gpu

MORE = {"text_rotate": ("eights", "row"), "text_weights": ("tiles", "single", "row"), "text_evict": ("one", "two"), "latent_append": (),
        "latent_decode": ("runs", "row"), "latent_attention": ("64", "128", "row")}


def zero(*shape):
    return torch.zeros(*shape, dtype=torch.float16, device="cuda")


def f32(*shape):
    return torch.zeros(*shape, device="cuda")


def ran(ctx, call):
    """The families and forms that a call runs, with how often."""
    names = [x for forms in (FORMS, MORE) for f in forms for x in [f] + [f"{f}_{y}" for y in forms[f]]]
    torch.cuda.synchronize()
    for n in names:
        ocrhip.probe_start(n)
    call()
    ctx.synchronize()
    got = {n: ocrhip.probe_stop(n)["calls"] for n in names}
    return {n: c for n, c in got.items() if c}


def one(*pairs):
    return {n: 1 for f, form in pairs for n in (f, f"{f}_{form}")}


def test_every_family_has_its_forms():
    assert set(MORE) == set(ocrhip.MORE_TEXT_FAMILIES)


@pytest.mark.parametrize("dim,first,rot,form", [(64, 0, 64, "eights"), (64, 8, 56, "eights"), (72, 0, 0, "eights"), (64, 4, 56, "row"), (64, 0, 36, "row"),
                                                (20, 0, 20, "row"), (1, 0, 0, "row")])
def test_rotation_forms(ctx, dim, first, rot, form):
    x, y = zero(9, 2, dim), zero(9, 2, dim)
    assert ran(ctx, lambda: ocrhip.rotate(ctx, x, i32(np.zeros((9, 2))), y, first=first, rot=rot, axes=(rot // 2, 0))) == one(("text_rotate", form))


@pytest.mark.parametrize("n,hq,dim,attends,weighs", [(40, 2, 64, "64", "tiles"), (9000, 16, 64, "128", "tiles"), (40, 2, 256, "128", "tiles"),
                                                    (40, 2, 15, "row", "row")])
def test_prompt_forms(ctx, n, hq, dim, attends, weighs):
    q, k, w = zero(n, hq, dim), zero(n, 1, dim), f32(1, 1, n)
    assert ran(ctx, lambda: ocrhip.attention(ctx, q, k, k, zero(n, hq, dim), weights=w)) == one(("text_attention", attends), ("text_weights", weighs))
    assert ran(ctx, lambda: ocrhip.attention(ctx, q, k, k, zero(n, hq, dim), weights=f32(1, 1, 0))) == one(("text_attention", attends))


@pytest.mark.parametrize("fmt,hq,dim,width,attends,weighs", [("f16", 1, 64, 13, "whole", None), ("f16", 16, 64, 13, "whole", None),
                                                            ("f16", 17, 64, 13, "whole", "single"), ("i8", 1, 64, 400, "parts", "single"),
                                                            ("i8", 1, 72, 4, "row", "row")])
def test_single_forms(ctx, fmt, hq, dim, width, attends, weighs):
    cache = ocrhip.KvCache(ctx, 2, 16, 1, dim, fmt)
    q, table, lens = zero(1, hq, dim), i32(np.zeros((1, width))), i32([0])
    w = f32(1, 1, 16 * width)
    want = one(("text_decode", attends), *([("text_weights", weighs)] if weighs else []))  # else the attention's workgroups add them up
    assert ran(ctx, lambda: cache.attend(table, lens, q, zero(1, hq, dim), weights=w)) == want


@pytest.mark.parametrize("fmt,dim,width,keep,form", [
    ("f16", 64, 3, 40, "one"), ("f16", 64, 40, 128, "one"), ("f16", 64, 40, 320, "two"), ("i8", 16, 300, 2048, "two"), ("i8", 16, 300, 1024, "one"),
    ("f16", 15, 3, 40, "one")])
def test_eviction_forms(ctx, fmt, dim, width, keep, form):
    cache = ocrhip.KvCache(ctx, 2, 16, 1, dim, fmt)
    w, h = f32(1, 1, 16 * width), i32(np.zeros((1, 1, 16 * width)))
    n, o = i32([0]), i32([0])
    assert ran(ctx, lambda: cache.evict(i32(np.full((1, width), -1)), n, n, w, h, keep, o)) == one(("text_evict", form))


@pytest.mark.parametrize("rank,rot,form", [(128, 32, "runs"), (512, 64, "runs"), (8, 0, "runs"), (100, 32, "row"), (64, 6, "row"), (64, 128, "row")])
def test_latent_forms(ctx, rank, rot, form):
    cache = ocrhip.LatentCache(ctx, 2, 16, rank, rot, "f16")
    t, n = i32([[0]]), i32([1])
    x, q, out = f32(1, rank + rot), zero(1, 2, rank + rot), zero(1, 2, rank)
    assert ran(ctx, lambda: cache.append(t, i32([0]), i32([0]), x)) == {"latent_append": 1}
    assert ran(ctx, lambda: cache.attend(t, n, q, out, scale=1.0)) == one(("latent_decode", form))


@pytest.mark.parametrize("n,heads,key,rot,value,form", [
    (1, 1, 8, 0, 8, "64"), (300, 12, 64, 32, 64, "64"), (5000, 12, 64, 32, 64, "128"), (40, 2, 128, 64, 128, "64"), (40, 2, 136, 0, 64, "row"),
    (40, 2, 64, 72, 64, "row"), (40, 2, 64, 6, 64, "row")])
def test_latent_prompt_forms(ctx, n, heads, key, rot, value, form):
    q, k, r, v = zero(n, heads, key + rot), zero(n, heads, key), zero(n, rot), zero(n, heads, value)
    call = lambda: ocrhip.latent_attention(ctx, q, k, r if rot else None, v, zero(n, heads, value))  # noqa: E731
    assert ran(ctx, call) == one(("latent_attention", form))


# ---- one step of everything, from the same start each time ---------------------------------------
def start(g):
    """Inputs of every operator (on the host), their sizes ragged."""
    s = {}
    s["x"], s["at"] = rn(g, 700, 3, 80).half(), torch.randint(0, 9000, (700, 3), generator=g).int()
    s["q"], s["k"], s["v"] = rn(g, 900, 8, 64).half(), rn(g, 900, 2, 64).half(), rn(g, 900, 2, 64).half()
    s["docs"], s["prefix"] = torch.tensor([0, 1, 130, 130, 870]).int(), torch.tensor([0, 50, 0, 300]).int()
    s["weights"] = torch.rand(4, 2, 740, generator=g)
    lens = [3000, 1, 517]
    t, pages = tables(g, lens, 16)
    s["table"], s["lens"], s["newest"] = torch.from_numpy(t), torch.tensor(lens).int(), torch.tensor([3100, 0, 516]).int()
    s["ck"], s["cv"] = rn(g, pages, 2, 16, 64).half(), rn(g, pages, 2, 16, 64).half()
    s["sq"], s["sw"] = rn(g, 3, 8, 64).half(), torch.rand(3, 2, 3000, generator=g)
    s["held"] = torch.full((3, 2, 3000), -1).int()
    s["pool"], s["lx"], s["lq"] = rn(g, pages, 16, 576).bfloat16(), rn(g, 3, 576), rn(g, 3, 40, 576).bfloat16()
    s["seq"], s["pos"] = torch.tensor([0, 1, 2]).int(), torch.tensor([2999, 0, 516]).int()
    s["pq"], s["pk"], s["pr"], s["pv"] = rn(g, 900, 4, 96).half(), rn(g, 900, 4, 64).half(), rn(g, 900, 32).half(), rn(g, 900, 4, 64).half()
    return s


def outputs(s, device):
    """The arrays on the device, with places for what the calls write."""
    d = {n: x.to(device) for n, x in s.items()}
    for n, like in (("rotated", "x"), ("out", "q"), ("single", "sq")):
        d[n] = torch.full_like(d[like], 7.0)
    d["absorbed"] = torch.full((3, 40, 512), 7.0, dtype=torch.bfloat16, device=device)
    d["expanded"] = torch.full((900, 4, 64), 7.0, dtype=torch.float16, device=device)
    d["left"] = torch.full((3,), -7, dtype=torch.int32, device=device)
    return d


def step(ctx, d):
    ocrhip.rotate(ctx, d["x"], d["at"], d["rotated"], first=8, rot=72, axes=(12, 12, 12), order="turns")
    ocrhip.attention(ctx, d["q"], d["k"], d["v"], d["out"], d["docs"], d["prefix"], weights=d["weights"], window=100)
    cache = ocrhip.KvCache(ctx, d["ck"].shape[0], 16, 2, 64, "f16", memory=(d["ck"], d["cv"], None, None))
    cache.attend(d["table"], d["lens"], d["sq"], d["single"], weights=d["sw"])
    cache.evict(d["table"], d["lens"], d["newest"], d["sw"], d["held"], 500, d["left"], first=4, recent=60)
    latent = ocrhip.LatentCache(ctx, d["pool"].shape[0], 16, 512, 64, "bf16", memory=d["pool"])
    latent.append(d["table"], d["seq"], d["pos"], d["lx"])
    latent.attend(d["table"], d["lens"], d["lq"], d["absorbed"], scale=0.05)
    ocrhip.latent_attention(ctx, d["pq"], d["pk"], d["pr"], d["pv"], d["expanded"], d["docs"], d["prefix"])


def alike(a, b):
    for n in a:
        assert torch.equal(a[n].cpu().view(torch.uint8), b[n].cpu().view(torch.uint8)), n


@pytest.fixture(scope="module")
def first(ctx):
    s = start(gen(77))
    d = outputs(s, "cuda")
    torch.cuda.synchronize()
    step(ctx, d)
    ctx.synchronize()
    assert (host(d["rotated"]) != 7).any() and (host(d["left"]) == [500, 1, 500]).all()
    assert (host(d["out"])[870:] == host(d["out"])[899]).all()  # rows of no document are all alike
    return s, d


def test_same_twice(ctx, first):
    s, d = first
    for _ in range(3):
        again = outputs(s, "cuda")
        torch.cuda.synchronize()
        step(ctx, again)
        ctx.synchronize()
        alike(again, d)


def test_without_the_native_module(ctx, first, monkeypatch):
    s, d = first
    again = outputs(s, "cuda")
    torch.cuda.synchronize()
    monkeypatch.setattr(text, "_native", lambda *a: False)
    step(ctx, again)
    ctx.synchronize()
    alike(again, d)


def test_other_streams(ctx, first):
    """Inputs that a stream of torch's is still making, outputs read there."""
    s, d = first
    stream = torch.cuda.Stream()
    fresh = outputs(s, "cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        busy = torch.zeros(4096, 4096, device="cuda")
        for _ in range(30):
            busy = busy @ busy
        again = {n: x + 0 for n, x in fresh.items()}
        ctx.acquire(stream.cuda_stream)
        step(ctx, again)
        ctx.release(stream.cuda_stream)
        got = {n: x + 0 for n, x in again.items()}
    stream.synchronize()
    alike(got, d)


def test_two_contexts_at_once(ctx, first):
    s, d = first
    other = ocrhip.Context()
    try:
        a, b = outputs(s, "cuda"), outputs(s, "cuda")
        torch.cuda.synchronize()
        step(ctx, a)
        step(other, b)
        ctx.synchronize()
        other.synchronize()
        alike(a, d)
        alike(b, d)
    finally:
        other.close()


def test_arrays_of_the_library(ctx, first):
    """The same calls on the library's own device memory, without torch."""
    s, d = first
    names = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32", torch.int32: "i32"}
    arrays = {}
    for n, x in outputs(s, "cpu").items():
        raw = x.contiguous().view(torch.uint8).numpy()
        b = ctx.alloc(raw.nbytes)
        b.upload(raw)
        arrays[n] = ocrhip.DeviceArray(b, tuple(x.shape), names[x.dtype])
    step(ctx, arrays)
    ctx.synchronize()
    for n, a in arrays.items():
        want = d[n].cpu().contiguous().view(torch.uint8).numpy().reshape(-1)
        assert np.array_equal(a.buffer.download(np.uint8, want.size), want), n


# ---- sizes ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,heads,rank", [(200, 16, 128), (131, 70, 512), (65, 1, 256)])
def test_many_sequences_of_latents(ctx, rows, heads, rank):
    """More rows than a wavefront scans at once, empty ones among them; a part of each of them is checked."""
    g = gen(rows)
    lens = [int(x) for x in (torch.rand(rows, generator=g) ** 3 * 900)]
    lens[7] = lens[64] = lens[rows - 1] = 0
    lens[rows - 2] = 2000
    w = rank + 32
    table, pages = tables(g, lens, 16)
    pool, q = rn(g, pages, 16, w).half(), rn(g, rows, heads, w).half()
    out = torch.full((rows, heads, rank), 9.0, dtype=torch.float16, device="cuda")
    cache = ocrhip.LatentCache(ctx, pages, 16, rank, 32, "f16", memory=pool.cuda())
    t, ls, qd = i32(table), i32(lens), q.cuda()
    torch.cuda.synchronize()
    cache.attend(t, ls, qd, out, scale=w ** -0.5)
    ctx.synchronize()
    got, held = host(out), pool.double().numpy()
    for r, n in enumerate(lens):
        c = np.concatenate([held[p] for p in table[r, : -(-n // 16)]])[:n] if n else np.zeros((0, w))
        want, size, top = plain.latent(q[r].double().numpy(), c, rank, w ** -0.5)
        close(got[r], want, size, top, EPS["f16"])


@pytest.mark.parametrize("rank,rot", [(512, 64), (512, 30)])
def test_latent_pool_past_32_bits(ctx, rank, rot):
    g, w, page = gen(4), rank + rot, 64
    pages = 2 ** 31 // (page * w) + 40  # values past 2^31, bytes past 2^32
    pool = torch.zeros(pages, page, w, dtype=torch.bfloat16, device="cuda")
    last = rn(g, 3, page, w).bfloat16()
    pool[-3:] = last.cuda()
    cache = ocrhip.LatentCache(ctx, pages, page, rank, rot, "bf16", memory=pool)
    t, n = i32([[pages - 1, pages - 3, pages - 2]]), 150
    x, q = rn(g, 1, w), rn(g, 1, 3, w).bfloat16()
    out, xd, qd = torch.zeros(1, 3, rank, dtype=torch.bfloat16, device="cuda"), x.cuda(), q.cuda()
    torch.cuda.synchronize()
    cache.append(t, i32([0]), i32([n - 1]), xd)
    cache.attend(t, i32([n]), qd, out, scale=0.04)
    ctx.synchronize()
    c = np.concatenate([last[k].double().numpy() for k in (2, 0, 1)])[:n]
    now = host(pool[-2, (n - 1) % page])
    assert np.array_equal(now[:rank], x[0, :rank].bfloat16().double().numpy())
    c[n - 1] = now
    want, size, top = plain.latent(q[0].double().numpy(), c, rank, 0.04)
    close(host(out)[0], want, size, top, EPS["bf16"])
    assert not pool[: pages - 3].any()


def test_eviction_past_32_bits(ctx):
    g, hk, page, dim = gen(5), 8, 64, 64
    pages = 2 ** 31 // (hk * page * dim) + 3
    k, v = (torch.zeros(pages, hk, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    old = rn(g, 2, hk, page, dim).half()
    k[-2:], v[-2:] = old.cuda(), -old.cuda()
    cache = ocrhip.KvCache(ctx, pages, page, hk, dim, "f16", memory=(k, v, None, None))
    w = torch.rand(1, hk, 128, generator=g)
    wd, held, left = w.cuda(), i32(np.full((1, hk, 128), -1)), i32([0])
    torch.cuda.synchronize()
    cache.evict(i32([[pages - 1, pages - 2]]), i32([128]), i32([127]), wd, held, 100, left, recent=5)
    ctx.synchronize()
    want = old.numpy().copy()
    for h in range(hk):
        for src, dst in plain.evict(w[0, h].numpy(), np.full(128, -1, np.int32), 128, 127, 100, 0, 5)[0]:
            want[1 - dst // page, h, dst % page] = want[1 - src // page, h, src % page]
    assert np.array_equal(k[-2:].cpu().numpy(), want) and np.array_equal(v[-2:].cpu().numpy(), -want)
    assert not k[:-2].any() and not v[:-2].any()


def test_refusals_reach_the_caller(ctx):
    x, at = zero(4, 2, 64), i32(np.zeros((4, 2)))
    with pytest.raises(ocrhip.OcrError, match="overlap"):
        ocrhip.rotate(ctx, x[:3], at[:3], x[1:])
    with pytest.raises(ocrhip.OcrError, match="axes of 33 pairs"):
        ocrhip.rotate(ctx, x, at, axes=(16, 17))
    q = zero(4, 2, 64)
    with pytest.raises(ocrhip.OcrError, match="weights overlap"):
        ocrhip.attention(ctx, q, x, x, zero(4, 2, 64), weights=q.view(torch.float32).view(-1)[:8].view(1, 2, 4))
    cache = ocrhip.KvCache(ctx, 3, 16, 2, 64, "f16")
    t, n = i32([[0, 1]]), i32([20])
    w, h = f32(1, 2, 32), i32(np.zeros((1, 2, 32)))
    with pytest.raises(ocrhip.OcrError, match="first and 20 recent"):
        cache.evict(t, n, i32([19]), w, h, 20, i32([0]), first=1, recent=20)
    with pytest.raises(ocrhip.OcrError, match="new lengths overlap"):
        cache.evict(t, n, i32([19]), w, h, 20, n)
    latent = ocrhip.LatentCache(ctx, 3, 16, 64, 16, "f16")
    y = zero(1, 2, 80)
    with pytest.raises(ocrhip.OcrError, match="overlap"):
        latent.attend(t, n, y, y[:, :, :64].as_strided((1, 2, 64), (128, 64, 1)), scale=1.0)
    with pytest.raises(ocrhip.OcrError, match="at most 512 and 128"):
        big = ocrhip.LatentCache(ctx, 1, 16, 576, 0, "f16")
        big.attend(t, n, zero(1, 1, 576), zero(1, 1, 576), scale=1.0)
    with pytest.raises(ocrhip.OcrError, match="overlap"):
        k = zero(5, 2, 64)
        ocrhip.latent_attention(ctx, k, k, None, zero(5, 2, 64), k)
