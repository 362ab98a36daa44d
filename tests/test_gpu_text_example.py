"""The example's decoder: what it writes, against the same model over whole sequences."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import text as plain

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "text_decoder.py")


def example():
    spec = importlib.util.spec_from_file_location("text_decoder", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def whole(ex, m, x, prefix):
    """Float32 logits of every position of one sequence, without cache or kernels."""
    n = len(x)
    x = x.float().cpu()
    norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    ranges = plain.key_ranges(n, None, [prefix])
    f = lambda w: w.float().cpu()  # noqa: E731
    for i in range(m.layers):
        q, k, v = plain.projections((norm(x) @ f(m.qkv[i])).numpy(), m.q_heads, m.heads, m.dim, np.arange(n), np.ones(m.dim), np.ones(m.dim),
                                    1e-6, m.dim, 1e4, "halves")
        o = plain.attention(q, k, v, ranges, m.dim ** -0.5)[0]
        x = x + torch.from_numpy(o).float().flatten(1) @ f(m.out[i])
        y = norm(x)
        x = x + (torch.nn.functional.silu(y @ f(m.gate[i])) * (y @ f(m.up[i]))) @ f(m.down[i])
    return norm(x) @ f(m.head)


@pytest.mark.parametrize("fmt,beams", [("f16", 3), ("i8", 4), ("e4m3", 2)])
def test_example_writes_what_the_model_says(ctx, fmt, beams):
    """Every beam's score is the sum of its tokens' log-probabilities by the whole-sequence model. A
    logit passes some ten roundings a layer (float16, half a step 2^-11; the cache's 2^-8 for int8 and
    2^-4 for e4m3 of the values, of which a softmax's mean keeps about an eighth), each relative to
    the largest logit; they are taken as independent of sign, four times their root sum."""
    ex = example()
    m = ex.Decoder(ctx)
    g = torch.Generator().manual_seed(5)
    counts, steps = [33, 16, 50], 9
    tokens = torch.randn(sum(counts), m.width, generator=g).to(m.dtype).cuda()
    text, scores = ex.write(m, tokens, counts, beams, steps, fmt)
    torch.cuda.synchronize()
    ctx.synchronize()
    text, scores, start = text.cpu(), scores.cpu(), 0
    held = {"f16": 2.0 ** -11, "i8": 2.0 ** -8, "e4m3": 2.0 ** -4}[fmt]
    for line, count in enumerate(counts):
        assert (scores[line, :-1] >= scores[line, 1:]).all()
        assert len({tuple(t) for t in text[line].tolist()}) == beams
        for beam in range(beams):
            t = text[line, beam].tolist()
            x = torch.cat([tokens[start: start + count].cpu(), m.embed.cpu()[torch.tensor(t[:-1])]])
            logits = whole(ex, m, x, count)[count - 1:]
            logp = torch.log_softmax(logits.double(), -1)
            want, top = 0.0, 0.0
            for s, c in enumerate(t):
                want += float(logp[s, c])
                top = max(top, float(logits[s].abs().max()))
                if c == ex.EOS:
                    assert all(c == ex.EOS for c in t[s:])
                    break
            tol = 4 * (10 * m.layers * 2.0 ** -22 + m.layers * (held / 8) ** 2 * 2) ** 0.5 * top * len(t) ** 0.5 * 2
            assert abs(float(scores[line, beam]) - want) <= tol, (line, beam, float(scores[line, beam]), want, tol)
        start += count
