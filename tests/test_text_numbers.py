"""Whole numbers that the C ABI's types do not hold are refused by the binding: ctypes would cut them."""
import pytest

import ocrhip


class _Context:
    """Stands for a context where the binding refuses before it calls the library."""
    device, handle = 0, None

    def alloc(self, nbytes):
        return _Buffer(self, nbytes)


class _Buffer:
    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes, self.ptr = ctx, nbytes, 4096


def _arr(shape, dtype):
    n = 64
    for v in shape:
        n *= max(v, 1)
    return ocrhip.DeviceArray(_Buffer(_Context(), 64 * n), shape, dtype)


@pytest.mark.parametrize("eos", [2 ** 31, 2 ** 32 + 2, 2 ** 64 + 2, -2 ** 31 - 1, -2 ** 32 + 2])
def test_end_tokens(eos):
    x, s, i = _arr((6, 10), "f32"), _arr((2, 3), "f32"), _arr((2, 3), "i32")
    with pytest.raises(ocrhip.OcrError, match="end token"):
        ocrhip.beam_select(_Context(), x, s, i, eos, s, i, i, i)


@pytest.mark.parametrize("rot", [2 ** 32, 2 ** 32 + 8, 2 ** 64 + 8, -2 ** 32 + 8])
def test_rotations(rot):
    ctx = _Context()
    cache = ocrhip.KvCache(ctx, 4, 16, 2, 8, "i8")
    with pytest.raises(ocrhip.OcrError, match="rotation"):
        cache.append(_arr((3, 2), "i32"), _arr((3,), "i32"), _arr((3,), "i32"), _arr((3, 64), "f32"), _arr((3, 4, 8), "f16"), rot=rot)


@pytest.mark.parametrize("sizes", [(2 ** 32 + 4, 16, 2, 8), (4, 2 ** 32 + 16, 2, 8), (4, 16, 2 ** 32 + 2, 8), (4, 16, 2, 2 ** 32 + 8)])
def test_cache_sizes(sizes):
    with pytest.raises(ocrhip.OcrError, match="cache"):
        ocrhip.KvCache(_Context(), *sizes, "f16")
