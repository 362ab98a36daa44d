"""Builds libocrhip.so for gfx950 in-tree: every HIP kernel file and host C++ file with hipcc,
in parallel, then one link; and the text decoder's calls on torch tensors with the host compiler. Run as `python -m ocrhip.build` from wgpu-ocr_amd/, or call build()."""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)  # wgpu-ocr_amd/
CSRC = os.path.join(ROOT, "csrc")
OBJ = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libocrhip.so")
CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# Packed FP32 is disabled: this pool has seen wrong results from some v_pk_* f32 forms.
DEVICE_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# Matrix products whose sums stay in ordinary registers: softmax kernels read and rescale them all
# the time, and each move to and from the accumulation registers is an instruction.
FILE_FLAGS = {f"text_{n}.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"] for n in ("attn", "decode", "expanded", "latent", "weights")}
COMMON = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function"]


def sources():
    out = []
    for d in (CSRC, os.path.join(CSRC, "kernels")):
        for f in sorted(os.listdir(d)):
            if f.endswith((".hip", ".cpp")):
                out.append(os.path.join(d, f))
    return out


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.relpath(src, CSRC).replace(os.sep, "_") + ".o")
    cmd = [HIPCC, *COMMON, *DEVICE_FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in (r.stderr or "").splitlines() if noise not in l)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{err}")
    if err.strip():
        sys.stderr.write(err + "\n")
    return obj


def _tensors() -> None:
    """ocrhip._tensors, the text decoder's calls on torch tensors (csrc/python/tensors.cpp). Left out where torch, the
    host compiler or a header is missing: the binding does without it."""
    import shutil
    import sysconfig

    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:  # the library needs none of it, and without torch nothing here calls it
        return

    out = os.path.join(PKG, "_tensors.so")
    tmp = out + f".tmp{os.getpid()}"
    include = [sysconfig.get_paths()["include"], *cpp_extension.include_paths()]
    missing = [h for h in ("Python.h", "torch/csrc/autograd/python_variable.h") if not any(os.path.exists(os.path.join(p, h)) for p in include)]
    if shutil.which(CXX) is None:
        missing.insert(0, CXX)
    if missing:
        if os.path.exists(out):  # of another build: it may not fit the library
            os.remove(out)
        sys.stderr.write(f"_tensors.so is left out, for want of {', '.join(missing)}: calls on torch tensors are checked in Python\n")
        return
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{p}" for p in include], os.path.join(CSRC, "python", "tensors.cpp"), "-o", tmp, "-L" + lib, "-ltorch_python",
           "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stderr}")
    if r.stderr.strip():
        sys.stderr.write(r.stderr)
    os.replace(tmp, out)


def build(jobs: int | None = None) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), max(1, min(16, os.cpu_count() or 4)))
    with cf.ThreadPoolExecutor(jobs) as ex:
        tensors = ex.submit(_tensors)
        objs = list(ex.map(_compile, srcs))
        tensors.result()
    tmp = LIB + f".tmp{os.getpid()}"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs, "-lz"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build())
