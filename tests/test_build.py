"""The C library stands without torch, and so does its build: a C++ host needs no Python module of it."""
import sys
import types

import pytest

from brodiffusion_b200 import _build


@pytest.fixture
def built(monkeypatch, tmp_path):
    """The library is up to date, the module for torch tensors is not there."""
    monkeypatch.setattr(_build, "is_stale", lambda: False)
    monkeypatch.setattr(_build, "BINDING_PATH", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(_build.subprocess, "run", lambda *a, **k: pytest.fail("a compiler was started"))
    return tmp_path


def test_without_torch(built, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert _build.build() == _build.LIB_PATH and _build.build_binding() is None and not list(built.iterdir())


def test_with_a_torch_without_cuda(built, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(version=types.SimpleNamespace(cuda=None)))
    assert _build.build() == _build.LIB_PATH and not list(built.iterdir())


def test_a_compiler_that_fails_is_reported(built, monkeypatch, capsys):
    monkeypatch.setattr(_build.subprocess, "run", lambda *a, **k: types.SimpleNamespace(returncode=1, stdout="", stderr="no such file"))
    with pytest.raises(RuntimeError, match="_binding.so"):
        _build.build()
    assert "no such file" in capsys.readouterr().err
