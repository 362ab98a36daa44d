"""Beam search over rows of very large logits: masks of the type's lowest value that leave nothing, and offsets
beside which the log of the sum vanishes. A row of equal logits gives each token -log(vocabulary)."""
import numpy as np
import pytest
import torch

import ocrhip
from oracle import text as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to("cuda")


def host(x):
    torch.cuda.synchronize()
    return x.cpu().double().numpy() if x.is_floating_point() else x.cpu().numpy()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("w,vocab", [(1, 97), (4, 97), (3, 2049), (8, 20001)])
@pytest.mark.parametrize("size", ["lowest", "largest", 1e20])
def test_rows_of_equal_logits(ctx, ty, w, vocab, size):
    info = torch.finfo(TYPES[ty])
    if size == 1e20 and ty == "f16":
        size = 1e4
    x = torch.full((2 * w, vocab), {"lowest": info.min, "largest": info.max}.get(size, size)).to(TYPES[ty])
    x[w:, ::2] = 0.5  # the second group: a mask that leaves half of them, if its value is the lowest
    scores = np.tile(-0.5 * np.arange(w, dtype=np.float32), (2, 1))
    out = [torch.zeros(2, w, device="cuda")] + [i32(np.zeros((2, w))) for _ in range(3)]
    sc, xs = torch.from_numpy(scores).cuda(), x.cuda()
    torch.cuda.synchronize()
    ocrhip.beam_select(ctx, xs, sc, None, None, *out)
    ctx.synchronize()
    got = [host(o) for o in out]
    # One rounding to float32, and the sum of the exponentials: 2^-21 of it.
    tol = lambda s: 2.0 ** -24 * np.abs(s) + 2.0 ** -21  # noqa: E731
    assert (np.abs(got[0][0] + np.log(vocab)) <= tol(got[0][0])).all()  # the first beam's first tokens
    assert (got[1][0] == 0).all() and np.array_equal(got[2][0], np.arange(w))
    want = plain.beam_select(host(x), scores, None, -1)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    assert (np.abs(got[0] - want[0]) <= tol(want[0])).all()
