"""Spans of value scales (tests/cpp/test_text_spans.cpp), on the CPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_text_spans(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ is not available")
    exe = str(tmp_path / "text_spans")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "wgpu-ocr_amd", "csrc"),
           os.path.join(ROOT, "tests", "cpp", "test_text_spans.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr
