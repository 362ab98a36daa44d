"""The rules and refusals of the text decoder's further operators on the CPU: the C ABI's checks
(tests/cpp/test_text_more.cpp) and the Python binding's."""
import ctypes
import os
import shutil
import subprocess

import pytest

import ocrhip
from ocrhip import text
from test_text_rules import CSRC, ROCM_INC, ROOT, _arr, _Context, _refuses


def test_more_rules(tmp_path):
    if shutil.which("g++") is None or not os.path.isdir(ROCM_INC):
        pytest.skip("g++ or the HIP headers are not available")
    exe = str(tmp_path / "text_more")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-D__HIP_PLATFORM_AMD__", "-I", CSRC, "-I", ROCM_INC,
           os.path.join(ROOT, "tests", "cpp", "test_text_more.cpp"), os.path.join(CSRC, "text_check.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr


def test_binding_refuses_axes():
    ctx = _Context()
    x, at = _arr((5, 4, 16), "f16"), _arr((5, 2), "i32")
    rot = ocrhip.rotate
    _refuses("inputs: f32, f16 or bf16|inputs: .* is wanted", rot, ctx, _arr((5, 4, 16), "i8"), at)
    _refuses("inputs: shape", rot, ctx, _arr((5, 64), "f16"), at, rot=16)
    _refuses("outputs: f16 is wanted", rot, ctx, x, at, _arr((5, 4, 16), "bf16"))
    _refuses("outputs: shape", rot, ctx, x, at, _arr((5, 4, 8), "f16"))
    _refuses("one after another", rot, ctx, _arr((5, 4, 16), "f16", (64, 1, 4)), at)
    _refuses("positions: i32", rot, ctx, x, _arr((5, 2), "f32"))
    _refuses("positions: shape", rot, ctx, x, _arr((4, 2), "i32"))
    _refuses("positions: shape", rot, ctx, x, _arr((5, 1, 2), "i32"))
    _refuses("equal parts", rot, ctx, x, _arr((5, 3), "i32"))
    _refuses("positions of 2 axes", rot, ctx, x, at, axes=(8,))
    _refuses("1 to 4", rot, ctx, x, _arr((5, 5), "i32"), axes=(1, 1, 1, 1, 4))
    _refuses("1 to 4", rot, ctx, x, at, axes=(-1, 9))
    _refuses("1 to 4", rot, ctx, x, at, axes=(2 ** 32, 8))
    _refuses("blocks", rot, ctx, x, at, order="rows")
    _refuses("ladder", rot, ctx, x, at, ladder="none")
    _refuses("halves", rot, ctx, x, at, pairs="thirds")
    _refuses("base", rot, ctx, x, at, theta=-1.0)
    _refuses("rotation of -2 values", rot, ctx, x, at, rot=-2)
    _refuses("from value -1", rot, ctx, x, at, first=-1, rot=16)
    cache = ocrhip.KvCache(ctx, 4, 16, 2, 16, "f16")
    t, i3, qkv, q = _arr((3, 2), "i32"), _arr((3,), "i32"), _arr((3, 128), "f16"), _arr((3, 4, 16), "f16")
    _refuses("without positions", cache.append, t, i3, i3, qkv, q, axes=(4, 4))
    _refuses("positions: shape", cache.append, t, i3, i3, qkv, q, at=_arr((4, 2), "i32"))
    _refuses("positions of 1 axes", cache.append, t, i3, i3, qkv, q, at=i3, axes=(4, 4))
    _refuses("blocks", cache.append, t, i3, i3, qkv, q, at=i3, order="mixed")


def test_binding_refuses_weights():
    ctx = _Context()
    q, kv, out, docs = _arr((5, 4, 8), "f16"), _arr((5, 2, 8), "f16"), _arr((5, 4, 8), "f16"), _arr((4,), "i32")
    att = ocrhip.attention
    _refuses("without weights", att, ctx, q, kv, kv, out, docs, window=3)
    for window in (0, -1, 2 ** 31):
        _refuses("window", att, ctx, q, kv, kv, out, docs, weights=_arr((3, 2, 5), "f32"), window=window)
    _refuses("weights: shape", att, ctx, q, kv, kv, out, docs, weights=_arr((2, 2, 5), "f32"))
    _refuses("weights: shape", att, ctx, q, kv, kv, out, docs, weights=_arr((3, 4, 5), "f32"))
    _refuses("weights: three dimensions", att, ctx, q, kv, kv, out, docs, weights=_arr((3, 2), "f32"))
    _refuses("weights: f32", att, ctx, q, kv, kv, out, docs, weights=_arr((3, 2, 5), "f16"))
    _refuses("weights: its values", att, ctx, q, kv, kv, out, docs, weights=_arr((3, 2, 5), "f32", (10, 1, 2)))
    cache = ocrhip.KvCache(ctx, 4, 16, 2, 8, "f16")
    t, lens = _arr((5, 2), "i32"), _arr((5,), "i32")
    _refuses("weights: shape", cache.attend, t, lens, q, out, weights=_arr((4, 2, 9), "f32"))
    _refuses("weights: shape", cache.attend, t, lens, q, out, weights=_arr((5, 4, 9), "f32"))
    _refuses("weights: f32", cache.attend, t, lens, q, out, weights=_arr((5, 2, 9), "i32"))


def test_binding_refuses_evictions():
    ctx = _Context()
    cache = ocrhip.KvCache(ctx, 8, 16, 2, 8, "f16")
    t, i3, n3, out = _arr((3, 2), "i32"), _arr((3,), "i32"), _arr((3,), "i32"), _arr((3,), "i32")
    w, h = _arr((3, 2, 32), "f32"), _arr((3, 2, 32), "i32")
    _refuses("page table", cache.evict, i3, i3, n3, w, h, 9, out)
    _refuses("lengths: shape", cache.evict, t, _arr((2,), "i32"), n3, w, h, 9, out)
    _refuses("newest", cache.evict, t, i3, _arr((2,), "i32"), w, h, 9, out)
    _refuses("weights: shape", cache.evict, t, i3, n3, _arr((3, 3, 32), "f32"), h, 9, out)
    _refuses("weights: f32", cache.evict, t, i3, n3, h, h, 9, out)
    _refuses("positions: shape", cache.evict, t, i3, n3, w, _arr((3, 2, 31), "i32"), 9, out)
    _refuses("positions: i32", cache.evict, t, i3, n3, w, w, 9, out)
    _refuses("the new lengths: shape", cache.evict, t, i3, n3, w, h, 9, _arr((4,), "i32"))
    _refuses("new weights: shape", cache.evict, t, i3, n3, w, h, 9, out, weights_out=_arr((3, 2, 16), "f32"))
    _refuses("new positions: i32", cache.evict, t, i3, n3, w, h, 9, out, held_out=w)
    for bad in ({"keep": -1}, {"keep": 2 ** 32}, {"keep": 9, "first": -1}, {"keep": 9, "recent": 2 ** 32}):
        _refuses("eviction", cache.evict, t, i3, n3, w, h, lens_out=out, **bad)


def test_binding_refuses_latent_calls():
    ctx = _Context()
    _refuses("f16 or bf16", ocrhip.LatentCache, ctx, 4, 16, 32, 8, "i8")
    _refuses("empty", ocrhip.LatentCache, ctx, 4, 0, 32, 8)
    _refuses("empty", ocrhip.LatentCache, ctx, 4, 16, 32, -2)
    _refuses("past 32 bits", ocrhip.LatentCache, ctx, 2 ** 32, 16, 32, 8, "f16", _arr((4, 16, 40), "f16"))
    _refuses("latent cache: shape", ocrhip.LatentCache, ctx, 4, 16, 32, 8, "f16", _arr((4, 16, 39), "f16"))
    _refuses("latent cache: f16", ocrhip.LatentCache, ctx, 4, 16, 32, 8, "f16", _arr((4, 16, 40), "bf16"))
    c = ocrhip.LatentCache(ctx, 4, 16, 32, 8, "f16")
    t, i3, x = _arr((3, 2), "i32"), _arr((3,), "i32"), _arr((3, 40), "f32")
    _refuses("page table", c.append, i3, i3, i3, x)
    _refuses("projections", c.append, t, i3, i3, _arr((3, 39), "f32"))
    _refuses("projections", c.append, t, i3, i3, _arr((3, 40), "f32", (1, 3)))
    _refuses("projections", c.append, t, i3, i3, _arr((3, 40), "i8"))
    _refuses("sequence numbers", c.append, t, _arr((2,), "i32"), i3, x)
    _refuses("positions: shape", c.append, t, i3, _arr((2,), "i32"), x)
    _refuses("norm: shape", c.append, t, i3, i3, x, norm=_arr((40,), "f32"))
    _refuses("outputs: f16", c.append, t, i3, i3, x, _arr((3, 40), "bf16"))
    _refuses("outputs: shape", c.append, t, i3, i3, x, _arr((3, 32), "f16"))
    _refuses("base", c.append, t, i3, i3, x, theta=0)
    _refuses("halves", c.append, t, i3, i3, x, pairs="odd")
    _refuses("without positions", c.append, t, i3, i3, x, axes=(2, 2))
    _refuses("equal parts", c.append, t, i3, i3, x, at=_arr((3, 3), "i32"))
    q, out = _arr((3, 4, 40), "f16"), _arr((3, 4, 32), "f16")
    _refuses("queries: shape", c.attend, t, i3, _arr((3, 4, 32), "f16"), out, 1.0)
    _refuses("queries: f16", c.attend, t, i3, _arr((3, 4, 40), "bf16"), out, 1.0)
    _refuses("outputs: shape", c.attend, t, i3, q, _arr((3, 4, 40), "f16"), 1.0)
    _refuses("lengths", c.attend, t, _arr((4,), "i32"), q, out, 1.0)
    _refuses("parents", c.fork, t, i3, _arr((2, 2), "i32"), i3, t, i3, i3)
    la = ocrhip.latent_attention
    q, k, r, v, out = _arr((5, 3, 12), "f16"), _arr((5, 3, 8), "f16"), _arr((5, 4), "f16"), _arr((5, 3, 6), "f16"), _arr((5, 3, 6), "f16")
    _refuses("queries: f16 or bf16", la, ctx, _arr((5, 3, 12), "f32"), k, r, v, out)
    _refuses("keys: f16 is wanted", la, ctx, q, _arr((5, 3, 8), "bf16"), r, v, out)
    _refuses("keys: shape", la, ctx, q, _arr((4, 3, 8), "f16"), r, v, out)
    _refuses("values: shape", la, ctx, q, k, r, _arr((5, 2, 6), "f16"), out)
    _refuses("outputs: shape", la, ctx, q, k, r, v, _arr((5, 3, 8), "f16"))
    _refuses("shared keys: rows", la, ctx, q, k, _arr((5, 5), "f16"), v, out)
    _refuses("shared keys: rows", la, ctx, q, k, _arr((5, 4), "bf16"), v, out)
    _refuses("no shared keys", la, ctx, q, k, None, v, out)
    _refuses("one after another", la, ctx, q, _arr((5, 3, 8), "f16", (24, 1, 3)), r, v, out)
    _refuses("documents: i32", la, ctx, q, k, r, v, out, _arr((2,), "f32"))
    _refuses("prefix: shape", la, ctx, q, k, r, v, out, _arr((3,), "i32"), _arr((3,), "i32"))


def test_null_arguments_are_errors():
    lib = ocrhip.lib()
    calls = {"ocr_kv_append_axes_device": 5, "ocr_rotate_device": 3, "ocr_attention_weights_device": 5, "ocr_decode_attention_weights_device": 6,
             "ocr_kv_evict_device": 4, "ocr_latent_append_device": 5, "ocr_latent_decode_device": 4, "ocr_latent_fork_device": 10,
             "ocr_latent_attention_device": 2}
    for name, n in calls.items():
        args = [None if t is not text.U32 else 0 for t in getattr(lib, name).argtypes]
        assert len(args) == n, name
        assert getattr(lib, name)(*args) == 1 and b"ctx" in lib.ocr_last_error(), name


@pytest.mark.parametrize("kind", ["ocr_axes", "ocr_rotate_args", "ocr_evict_args", "ocr_latent_cache", "ocr_latent_append_args",
                                  "ocr_latent_decode_args", "ocr_latent_attention_args"])
def test_structures_are_the_headers(kind, tmp_path):
    """The binding's fields lie where the C compiler puts the header's."""
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not available")
    fields = [f[0] for f in getattr(text, kind)._fields_]
    src = tmp_path / "at.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ocrhip.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof({kind}, {f}));\n' for f in fields) + f'printf("%zu", sizeof({kind})); return 0; }}\n')
    exe = str(tmp_path / "at")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    t = getattr(text, kind)
    assert got == [getattr(t, f).offset for f in fields] + [ctypes.sizeof(t)]
