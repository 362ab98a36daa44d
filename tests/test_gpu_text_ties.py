"""Beam search where scores tie: scores that absorb the logits (a beam masked by a large finite
score), logits that vanish beside the log-sum. Against float64 (oracle/text.py): equal scores go to
the lower beam * vocab + token, and every place is written."""
import numpy as np
import pytest
import torch

import ocrhip
from oracle import text as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOWEST = float(np.finfo(np.float32).min)
SHAPES = [(1, 97), (2, 97), (3, 5), (4, 97), (5, 2048), (8, 5000), (32, 97), (32, 2049), (32, 20001), (4, 131072)]  # beams, vocabulary


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to("cuda")


def host(x):
    torch.cuda.synchronize()
    return x.cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()


def select(ctx, x, scores, finished=None, eos=None):
    g, w = scores.shape
    out = [torch.full((g, w), 7.0, device="cuda")] + [i32(np.full((g, w), -5)) for _ in range(3)]
    sc, fin = torch.from_numpy(scores.astype(np.float32)).cuda(), None if finished is None else i32(finished)
    torch.cuda.synchronize()
    ocrhip.beam_select(ctx, x, sc, fin, eos, *out)
    ctx.synchronize()
    return [host(o) for o in out]


def beam(ctx, x, scores, finished=None, eos=None):
    got = select(ctx, x, scores, finished, eos)
    want = plain.beam_select(host(x), scores.astype(np.float32), finished, -1 if eos is None else eos)
    for a, b in zip(got[1:], want[1:]):
        assert np.array_equal(a, b), (a, b)
    fine = np.isfinite(want[0])
    assert np.array_equal(got[0][~fine], want[0][~fine])
    # One rounding to float32, and the sum of the exponentials: 2^-21 of it.
    assert (np.abs(got[0][fine] - want[0][fine]) <= 2.0 ** -24 * np.abs(want[0][fine]) + 2.0 ** -21).all()


def logits(w, vocab, ty, groups=3):
    g = torch.Generator().manual_seed(w * 1000003 + vocab)
    return (torch.randn(groups * w, vocab, generator=g) * 3).to(TYPES[ty])


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("w,vocab", SHAPES)
@pytest.mark.parametrize("dead", [-1e20, -1e30, LOWEST, -LOWEST])
def test_scores_that_absorb_logits(ctx, ty, w, vocab, dead):
    """All beams, one, or all but the first hold a score beside which a logit is nothing."""
    x = logits(w, vocab, ty)
    scores = np.full((3, w), dead)
    scores[1] = -np.arange(w) * 0.5
    scores[1, w // 2] = dead
    scores[2, 0] = 0.0
    beam(ctx, x.cuda(), scores)
    beam(ctx, x.cuda(), scores, (np.arange(3 * w).reshape(3, w) % 5 == 3).astype(np.int32), min(2, vocab - 1))


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("w,vocab", SHAPES)
@pytest.mark.parametrize("allowed", [1, 2, 7])
@pytest.mark.parametrize("dead", [-1e30, LOWEST])
def test_first_step_of_few_allowed_tokens(ctx, ty, w, vocab, allowed, dead):
    """A first step whose first beam has fewer tokens that count than there are beams: the others'
    fill the places that are left."""
    x = logits(w, vocab, ty)
    keep = torch.randint(0, vocab, (allowed,), generator=torch.Generator().manual_seed(allowed))
    masked = torch.full_like(x, -float("inf"))
    masked[:, keep] = x[:, keep]
    scores = np.full((3, w), dead)
    scores[:, 0] = 0.0
    beam(ctx, masked.cuda(), scores)
    scores[1, 1:] = -np.inf
    beam(ctx, masked.cuda(), scores)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("w,vocab", SHAPES)
@pytest.mark.parametrize("size", [1e-17, 1e-30, 1e-42])
def test_logits_that_vanish(ctx, ty, w, vocab, size):
    """Logits all different and all nothing beside the log-sum, some of them beside larger ones."""
    x = logits(w, vocab, "f32") * size
    x[w:2 * w, ::3] = -2.5
    x[2 * w:, vocab // 2] = 1.25
    beam(ctx, x.to(TYPES[ty]).cuda(), np.tile(-0.25 * np.arange(w), (3, 1)))


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("w,vocab", [(4, 97), (32, 97), (8, 20001)])
def test_scores_that_absorb_some(ctx, ty, w, vocab):
    """Scores of 10^9 to 10^12, whose float64 steps are of the logits' size: which logits tie depends on
    the log-sum's last bits, but every place holds a continuation of its own, in the scores' order."""
    x = logits(w, vocab, ty)
    scores = np.array([[-1e9], [-1e10], [-1e12]]) * np.ones((3, w))
    s, p, t, f = select(ctx, x.cuda(), scores, None, 2)
    assert ((p >= 0) & (p < w) & (t >= 0) & (t < vocab)).all() and np.array_equal(f, (t == 2).astype(np.int32))
    assert (np.diff(s, axis=1) <= 0).all()
    for g in range(3):
        assert len(set(zip(p[g], t[g]))) == w
    assert (np.abs(s - scores) <= 2.0 ** -23 * np.abs(scores)).all()
