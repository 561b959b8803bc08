"""build.py without a GPU: what is built, in which order, and what may be missing."""

from __future__ import annotations

import importlib
import subprocess

import pytest

from conftest import PKG_NAME


@pytest.fixture
def b():
    return importlib.import_module(PKG_NAME + ".build")


@pytest.fixture
def calls(b, monkeypatch, tmp_path):
    """Both outputs in a folder of their own, nothing compiled: the commands' programs, in order."""
    ran = []

    def run(cmd, **kw):
        ran.append("nvcc" if b.SRC in cmd else "g++")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b, "OUT", str(tmp_path / "libbsgemm.so"))
    monkeypatch.setattr(b, "BIND_OUT", str(tmp_path / "_native.so"))
    monkeypatch.setattr(b.subprocess, "run", run)
    return ran


def test_library_first(b, calls):
    assert b.build(force=True) == b.OUT
    assert calls == ["nvcc", "g++"]


@pytest.mark.parametrize("err", [ImportError("No module named 'torch'"), FileNotFoundError("g++")])
def test_library_without_host_path(b, calls, monkeypatch, capsys, err):
    """A host with nvcc alone gets the library; the message names what is missing."""
    def fail(force=False):
        raise err
    monkeypatch.setattr(b, "build_native", fail)
    assert b.build(force=True) == b.OUT and calls == ["nvcc"]
    assert str(err) in capsys.readouterr().err


def test_compile_error_is_raised(b, calls, monkeypatch):
    """An error in the host path's own source is no missing tool; the library is there by then."""
    def fail(force=False):
        raise RuntimeError("g++ failed (1)")
    monkeypatch.setattr(b, "build_native", fail)
    with pytest.raises(RuntimeError, match="failed"):
        b.build(force=True)
    assert calls == ["nvcc"]


def test_host_path_follows_torch(b, calls, monkeypatch):
    """Another torch or Python than the one it was built for builds the host path again; the same one does not."""
    b.build_native()
    b.build_native()
    assert calls == ["g++"]
    monkeypatch.setattr(b, "native_versions", lambda: "torch 9.9.9 cxx11_abi 1 python cpython-399")
    b.build_native()
    b.build_native()
    assert calls == ["g++", "g++"]
