"""The text decoder's rules and refusals on the CPU: the C ABI's checks (tests/cpp/test_text_rules.cpp)
and the Python binding's."""
import ctypes
import os
import shutil
import subprocess

import pytest

import ocrhip
from ocrhip import text

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "wgpu-ocr_amd", "csrc")
ROCM_INC = "/opt/rocm/include"


def test_text_rules(tmp_path):
    if shutil.which("g++") is None or not os.path.isdir(ROCM_INC):
        pytest.skip("g++ or the HIP headers are not available")
    exe = str(tmp_path / "text_rules")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-D__HIP_PLATFORM_AMD__", "-I", CSRC, "-I", ROCM_INC,
           os.path.join(ROOT, "tests", "cpp", "test_text_rules.cpp"), os.path.join(CSRC, "text_check.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr


class _Context:
    """Stands for a context where the binding refuses before it calls the library."""
    device, handle = 0, None

    def alloc(self, nbytes):
        return _Buffer(self, nbytes)


class _Buffer:
    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes, self.ptr = ctx, nbytes, 4096


def _arr(shape, dtype, strides=None, ctx=None):
    ctx = ctx or _Context()
    n = 64
    for v in shape:
        n *= max(v, 1)
    return ocrhip.DeviceArray(_Buffer(ctx, 64 * n), shape, dtype, strides)


def _refuses(part, fn, *args, **kw):
    with pytest.raises(ocrhip.OcrError, match=part):
        fn(*args, **kw)


def test_binding_refuses_arrays():
    ctx = _Context()
    _refuses("does not fit", ocrhip.DeviceArray, _Buffer(ctx, 63), (4, 4), "f32")
    _refuses("does not fit", ocrhip.DeviceArray, _Buffer(ctx, 64), (4, 4), "f32", (5, 1))
    _refuses("type of", ocrhip.DeviceArray, _Buffer(ctx, 64), (4, 4), "f64")
    _refuses("strides", ocrhip.DeviceArray, _Buffer(ctx, 64), (4, 4), "f32", (-4, 1))
    q, kv, out = _arr((5, 4, 8), "f16"), _arr((5, 2, 8), "f16"), _arr((5, 4, 8), "f16")
    att = ocrhip.attention
    _refuses("queries: f16 or bf16", att, ctx, _arr((5, 4, 8), "f32"), kv, kv, out)
    _refuses("keys: f16 is wanted", att, ctx, q, _arr((5, 2, 8), "bf16"), kv, out)
    _refuses("values: shape", att, ctx, q, kv, _arr((5, 1, 8), "f16"), out)
    _refuses("keys: shape", att, ctx, q, _arr((4, 2, 8), "f16"), kv, out)
    _refuses("outputs: shape", att, ctx, q, kv, kv, _arr((5, 4, 16), "f16"))
    _refuses("one after another", att, ctx, _arr((5, 4, 8), "f16", (32, 1, 4)), kv, kv, out)
    _refuses("offsets", att, ctx, q, kv, kv, out, _arr((1, 2), "i32"))
    _refuses("documents: i32", att, ctx, q, kv, kv, out, _arr((2,), "f32"))
    _refuses("prefix: shape", att, ctx, q, kv, kv, out, _arr((3,), "i32"), _arr((3,), "i32"))
    _refuses("slopes: shape", att, ctx, q, kv, kv, out, slopes=_arr((2,), "f32"))
    import numpy as np
    _refuses("not an array in the memory", att, ctx, np.zeros((5, 4, 8), np.float16), kv, kv, out)
    import torch
    _refuses("not an array in the memory", att, ctx, torch.zeros(5, 4, 8, dtype=torch.float16), kv, kv, out)
    other = _Context()
    other.device = 1
    _refuses("device 0", att, ctx, _arr((5, 4, 8), "f16", ctx=other), kv, kv, out)


def test_binding_refuses_cache_calls():
    ctx = _Context()
    _refuses("f16, bf16, i8 or e4m3", ocrhip.KvCache, ctx, 4, 16, 2, 8, "f32")
    _refuses("empty", ocrhip.KvCache, ctx, 4, 0, 2, 8)
    c = ocrhip.KvCache(ctx, 4, 16, 2, 8, "i8")
    mem = (c.k, c.v, c.k_scale, c.v_scale)
    _refuses("needs scales", ocrhip.KvCache, ctx, 4, 16, 2, 8, "i8", (c.k, c.v, None, None))
    _refuses("cache keys: shape", ocrhip.KvCache, ctx, 5, 16, 2, 8, "i8", (c.k, c.v, _arr((5, 2, 16), "f32"), _arr((5, 2, 16), "f32")))
    _refuses("cache keys: bf16", ocrhip.KvCache, ctx, 4, 16, 2, 8, "bf16", mem)
    table, i3 = _arr((3, 2), "i32"), _arr((3,), "i32")
    q, qkv = _arr((3, 4, 8), "f16"), _arr((3, 64), "f32")
    _refuses("page table: shape", c.append, i3, i3, i3, qkv, q)
    _refuses("page table: its values", c.append, _arr((3, 2), "i32", (1, 3)), i3, i3, qkv, q)
    _refuses("projections", c.append, table, i3, i3, _arr((3, 63), "f32"), q)
    _refuses("projections", c.append, table, i3, i3, _arr((3, 64), "f32", (1, 3)), q)
    _refuses("queries: shape", c.append, table, i3, i3, qkv, _arr((3, 4, 9), "f16"))
    _refuses("queries: its values", c.append, table, i3, i3, qkv, _arr((3, 4, 8), "f16", (40, 8, 1)))
    _refuses("positions: shape", c.append, table, i3, _arr((2,), "i32"), qkv, q)
    _refuses("halves", c.append, table, i3, i3, qkv, q, pairs="thirds")
    _refuses("base", c.append, table, i3, i3, qkv, q, theta=0)
    _refuses("q_norm: shape", c.append, table, i3, i3, qkv, q, q_norm=_arr((4,), "f32"))
    _refuses("keys: f16 is wanted", c.append, table, i3, i3, qkv, q, k=_arr((3, 2, 8), "bf16"))
    _refuses("keys: shape", c.read, table, i3, _arr((3, 9, 2, 7), "f16"), _arr((3, 9, 2, 8), "f16"))
    _refuses("values: f16 is wanted", c.read, table, i3, _arr((3, 9, 2, 8), "f16"), _arr((3, 9, 2, 8), "bf16"))
    _refuses("lengths", c.attend, table, _arr((2,), "i32"), q, q)
    _refuses("queries: shape", c.attend, table, i3, _arr((2, 4, 8), "f16"), q)
    _refuses("parents", c.fork, table, i3, _arr((2, 2), "i32"), i3, table, i3, i3)
    _refuses("new table: shape", c.fork, table, i3, _arr((1, 3), "i32"), i3, _arr((3, 3), "i32"), i3, i3)


def test_binding_refuses_beams():
    ctx = _Context()
    x, s, i = _arr((6, 10), "f32"), _arr((2, 3), "f32"), _arr((2, 3), "i32")
    _refuses("logits", ocrhip.beam_select, ctx, _arr((5, 10), "f32"), s, i, 2, s, i, i, i)
    _refuses("logits", ocrhip.beam_select, ctx, _arr((6, 10), "i8"), s, i, 2, s, i, i, i)
    _refuses("logits", ocrhip.beam_select, ctx, _arr((6, 10), "f32", (1, 6)), s, i, 2, s, i, i, i)
    _refuses("scores", ocrhip.beam_select, ctx, x, _arr((6,), "f32"), i, 2, s, i, i, i)
    _refuses("parents: i32", ocrhip.beam_select, ctx, x, s, i, 2, s, s, i, i)


def test_null_context_is_an_error():
    args = text.ocr_attention_args()
    assert ocrhip.lib().ocr_attention_device(None, ctypes.byref(args)) == 1
    assert b"ctx" in ocrhip.lib().ocr_last_error()
    assert ocrhip.lib().ocr_stream_acquire(None, None) == 1
