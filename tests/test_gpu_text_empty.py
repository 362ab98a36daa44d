"""Calls of torch over no sequences and no tokens: empty tensors have no address, nothing is done."""
import pytest
import torch

import ocrhip

pytestmark = pytest.mark.gpu


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("width", [0, 3])
def test_no_sequences(ctx, width):
    cache = ocrhip.KvCache(ctx, 2, 16, 1, 64, "i8")
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    table, none = i32(0, width), i32(0)
    cache.append(table, none, none, half(0, 4 * 64), half(0, 2, 64))
    cache.read(table, none, half(0, 5, 1, 64), half(0, 5, 1, 64))
    cache.attend(table, none, half(0, 2, 64), half(0, 2, 64))
    cache.fork(table, none, i32(0, 4), none, i32(0, width), none, none)
    f = torch.zeros(0, 4, device="cuda")
    ocrhip.beam_select(ctx, torch.zeros(0, 97, device="cuda"), f, None, None, f, i32(0, 4), i32(0, 4))
    # Tokens of no sequence have queries all the same.
    x = torch.randn(3, 4 * 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    q = half(3, 2, 64)
    torch.cuda.synchronize()
    cache.append(table, i32(3), i32(3), x, q, rot=0)
    ctx.synchronize()
    assert torch.equal(q, x[:, :128].view(3, 2, 64))
