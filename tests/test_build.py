"""Building the C module of the dense operators' calls: it is optional, and goes with the torch it
was built against."""
import importlib
import os
import subprocess
import sys

import pytest

import mlx_rs_b200
from mlx_rs_b200 import ops


@pytest.fixture
def build(monkeypatch, tmp_path):
    """build.py with the C module going to a folder of its own; the library stands built."""
    mlx_rs_b200.library()
    b = importlib.import_module("mlx_rs_b200.build")
    monkeypatch.setattr(b, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(b, "CALLS_FOR", str(tmp_path / "calls.for"), raising=False)
    return b


@pytest.mark.parametrize("command", [["false"], ["no-such-compiler"]])
def test_the_library_builds_without_the_c_module(build, monkeypatch, command, capsys):
    open(build.CALLS, "w").close()
    os.utime(build.CALLS, (0, 0))  # an old one, which no longer fits
    monkeypatch.setattr(build, "calls_command", lambda src: command)
    assert build.build() == build.LIB
    assert not os.path.exists(build.CALLS)
    assert "_calls" in capsys.readouterr().err


def test_the_c_module_is_built_again_for_another_torch(build, monkeypatch):
    runs = []

    def command(src):
        runs.append(src)
        return [sys.executable, "-c", f"open({build.CALLS!r}, 'w').close()"]
    monkeypatch.setattr(build, "calls_command", command)
    build.build()
    build.build()
    assert len(runs) == 1
    monkeypatch.setattr(build, "calls_for", lambda: "another torch")
    build.build()
    assert len(runs) == 2


def test_a_c_module_of_another_torch_is_not_used(monkeypatch):
    assert ops.load_calls() is not None
    monkeypatch.setattr(sys.modules["mlx_rs_b200._calls"], "torch_version", "1.0.0")
    with pytest.warns(UserWarning, match="1.0.0"):
        assert ops.load_calls() is None
    monkeypatch.undo()
    assert ops.load_calls() is not None


def test_a_c_module_built_after_the_import_is_used():
    """A fresh checkout: ops is imported, then the first call builds the libraries."""
    code = """
import mlx_rs_b200
from mlx_rs_b200 import _lib, build, ops
import os, sys, importlib
real = build.CALLS
assert ops._calls is not None
ops._calls = None                      # as where there was no C module at the import
sys.modules.pop("mlx_rs_b200._calls", None)
path, _lib.library_path, _lib._lib = _lib.library_path, "/nonexistent", None
def built():
    _lib.library_path = path
    return path
build.build = built
_lib.library()
assert ops._calls is not None
print("loaded")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=120)
    assert "loaded" in r.stdout, r.stderr[-1500:]
