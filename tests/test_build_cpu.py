"""The build of the Python binding: left out where torch or the headers are
not installed, with the library as it was for users of the C ABI."""
import os
import shutil
import subprocess
import sys

import pytest

from luisaml_amd import build, capi


@pytest.fixture
def stale(tmp_path, monkeypatch):
    """A binding of an earlier build, in a place of its own."""
    path = tmp_path / "_binding.so"
    path.write_bytes(b"old")
    monkeypatch.setattr(build, "BINDING", str(path))
    return path


def test_without_torch(stale, monkeypatch, capfd):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert not build._build_binding()
    assert not stale.exists() and "torch not found" in capfd.readouterr().err


def test_without_headers(stale, monkeypatch, capfd, tmp_path):
    from torch.utils import cpp_extension
    with monkeypatch.context() as m:
        m.setattr(cpp_extension, "include_paths", lambda *a, **k: [str(tmp_path)])
        assert not build._build_binding()
    assert "torch's headers not found" in capfd.readouterr().err and not stale.exists()
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert not build._build_binding()
    assert "Python's headers not found" in capfd.readouterr().err


def test_compiler(stale, monkeypatch):
    """CXX, else g++, else hipcc; a failing one is an error."""
    used = []

    def run(cmd, **kw):
        used.append(cmd[0])
        return subprocess.CompletedProcess(cmd, 1, "", "no")
    monkeypatch.setattr(build.subprocess, "run", run)
    for env, which in ((dict(CXX="mine"), "/usr/bin/g++"), ({}, "/usr/bin/g++"), ({}, None)):
        monkeypatch.delenv("CXX", raising=False)
        for k, v in env.items():
            monkeypatch.setenv(k, v)
        monkeypatch.setattr(shutil, "which", lambda name: which)
        with pytest.raises(RuntimeError, match="binding failed"):
            build._build_binding()
    assert used == ["mine", "/usr/bin/g++", build.HIPCC]


def test_capi_says_what_is_missing(monkeypatch, tmp_path):
    capi.lib()
    monkeypatch.setattr(capi, "_native", None)
    monkeypatch.setattr(capi, "HERE", str(tmp_path))
    with pytest.raises(RuntimeError, match="_binding.so is not built"):
        capi._binding()
    assert os.path.exists(capi.LIB_PATH)
