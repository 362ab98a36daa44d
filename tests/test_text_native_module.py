"""The native module for calls on torch tensors is a shorter way, not a condition: the library builds
without a host compiler or Python's headers, and calls without the module go through the binding's checks."""
import os
import sys
import sysconfig

import pytest

import ocrhip
from ocrhip import build, text


class _Context:
    device, handle = 0, None

    def alloc(self, nbytes):
        return _Buffer(self, nbytes)


class _Buffer:
    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes, self.ptr = ctx, nbytes, 4096


@pytest.mark.parametrize("missing", ["compiler", "headers"])
def test_build_without(monkeypatch, tmp_path, capsys, missing):
    pytest.importorskip("torch")
    monkeypatch.setattr(build, "PKG", str(tmp_path))
    old = tmp_path / "_tensors.so"
    old.write_bytes(b"of another build")
    if missing == "compiler":
        monkeypatch.setattr(build, "CXX", str(tmp_path / "no-such-compiler"))
    else:
        paths = dict(sysconfig.get_paths(), include=str(tmp_path))
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: paths)
    build._tensors()
    assert not os.path.exists(old)  # one of another build may not fit the library
    assert "_tensors" in capsys.readouterr().err


def test_calls_without(monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(text, "_tensors", None)
    monkeypatch.delattr(ocrhip, "_tensors", raising=False)
    monkeypatch.setitem(sys.modules, "ocrhip._tensors", None)
    ctx = _Context()
    q, kv = (ocrhip.DeviceArray(_Buffer(ctx, 4096), (5, h, 8), "f16") for h in (4, 2))
    with pytest.warns(RuntimeWarning, match="_tensors"):
        with pytest.raises(ocrhip.OcrError, match="ctx"):  # every check passed, and the library has no context
            ocrhip.attention(ctx, q, kv, kv, q)
    with pytest.raises(ocrhip.OcrError, match="keys: shape"):
        ocrhip.attention(ctx, q, ocrhip.DeviceArray(_Buffer(ctx, 4096), (4, 2, 8), "f16"), kv, q)
