"""Which kernel each of the text decoder's calls runs: the rules on sizes and alignment, by the probe's names."""
import pytest
import torch

import ocrhip

pytestmark = pytest.mark.gpu

FORMS = {"text_append": ("eights", "row"), "text_read": ("eights", "row"), "text_attention": ("64", "128", "row"),
         "text_decode": ("whole", "parts", "row"), "text_fork": ("pieces", "bytes"), "beam_select": ("one", "two")}


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16, device="cuda")


def ran(ctx, call):
    """The families and forms that a call runs, with how often."""
    names = list(ocrhip.TEXT_FAMILIES) + [f"{f}_{x}" for f in ocrhip.TEXT_FAMILIES for x in FORMS[f]]
    torch.cuda.synchronize()
    for n in names:
        ocrhip.probe_start(n)
    call()
    ctx.synchronize()
    got = {n: ocrhip.probe_stop(n)["calls"] for n in names}
    return {n: c for n, c in got.items() if c}


def one(family, form):
    return {family: 1, f"{family}_{form}": 1}


def test_every_family_has_its_forms():
    assert set(FORMS) == set(ocrhip.TEXT_FAMILIES)


@pytest.mark.parametrize("fmt,dim,rot,pairs,append,read", [
    ("i8", 64, 64, "halves", "eights", "eights"), ("f16", 72, 64, "halves", "eights", "eights"), ("e4m3", 64, 4, "adjacent", "eights", "eights"),
    ("f16", 64, 36, "halves", "row", "eights"), ("i8", 20, 20, "halves", "row", "row"), ("bf16", 1, 0, "halves", "row", "row")])
def test_cache(ctx, fmt, dim, rot, pairs, append, read):
    cache = ocrhip.KvCache(ctx, 2, 16, 1, dim, fmt)
    t = i32(1, 2)
    assert ran(ctx, lambda: cache.append(t, i32(3), i32(3), half(3, 4 * dim), half(3, 2, dim), rot=rot, pairs=pairs)) == one("text_append", append)
    assert ran(ctx, lambda: cache.read(t, i32(1), half(1, 5, 1, dim), half(1, 5, 1, dim))) == one("text_read", read)


@pytest.mark.parametrize("n,hq,dim,form", [
    (1, 1, 8, "64"), (109, 8, 64, "64"), (6144, 16, 64, "64"), (6145, 16, 64, "128"), (2048, 16, 128, "64"), (2049, 16, 128, "128"), (10, 2, 256, "128"),
    (10, 2, 15, "row"), (10, 2, 4, "row")])
def test_prompts(ctx, n, hq, dim, form):
    q, k = half(n, hq, dim), half(n, 1, dim)
    assert ran(ctx, lambda: ocrhip.attention(ctx, q, k, k, half(n, hq, dim))) == one("text_attention", form)


def test_prompts_that_do_not_lie_on_pieces(ctx):
    x = half(10 * 72 + 8)
    on, off, odd = x[8:648].view(10, 64), x[1:641].view(10, 64), x[8:728].view(10, 72)[:, :64]
    at = lambda y: y.unflatten(1, (1, 64))  # noqa: E731
    for y, form in ((on, "64"), (off, "row"), (odd, "64")):
        assert ran(ctx, lambda: ocrhip.attention(ctx, at(y), at(y), at(y), half(10, 1, 64))) == one("text_attention", form)


@pytest.mark.parametrize("fmt,rows,hk,dim,width,form", [
    ("f16", 1, 8, 64, 13, "whole"), ("i8", 1, 8, 64, 16, "whole"), ("i8", 1, 8, 64, 17, "parts"), ("i8", 144, 4, 128, 44, "whole"),
    ("e4m3", 4, 8, 128, 2000, "parts"), ("i8", 1, 1, 72, 400, "row"), ("f16", 1, 1, 72, 400, "parts"), ("f16", 1, 1, 15, 4, "row")])
def test_single_tokens(ctx, fmt, rows, hk, dim, width, form):
    cache = ocrhip.KvCache(ctx, 2, 16, hk, dim, fmt)
    q, table, lens = half(rows, hk, dim), i32(rows, width), i32(rows)
    assert ran(ctx, lambda: cache.attend(table, lens, q, half(rows, hk, dim))) == one("text_decode", form)


@pytest.mark.parametrize("fmt,dim,form", [("f16", 8, "pieces"), ("i8", 8, "bytes"), ("i8", 16, "pieces"), ("f16", 15, "bytes")])
def test_forks(ctx, fmt, dim, form):
    cache = ocrhip.KvCache(ctx, 8, 16, 1, dim, fmt)
    t, n = i32(4, 2), i32(4)
    assert ran(ctx, lambda: cache.fork(t, n, i32(2, 2), i32(4), i32(4, 2), i32(4), i32(4))) == one("text_fork", form)


@pytest.mark.parametrize("vocab,form", [(97, "one"), (2048, "one"), (2049, "two")])
def test_beams(ctx, vocab, form):
    s, x = torch.zeros(2, 3, device="cuda"), torch.zeros(6, vocab, device="cuda")
    assert ran(ctx, lambda: ocrhip.beam_select(ctx, x, s, None, None, torch.zeros(2, 3, device="cuda"), i32(2, 3), i32(2, 3))) == one("beam_select", form)
