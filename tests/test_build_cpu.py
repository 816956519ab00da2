"""The build's order and its needs, with the compilers replaced."""
import os
import subprocess
import sys
import types

import pytest

from cpp_inference_train_engine_b200 import build as B


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    """Records the commands; every one writes its output. The outputs live in tmp_path."""
    ran = []

    def run(command, **kw):
        ran.append(os.path.basename(command[0]))
        with open(command[command.index("-o") + 1], "w") as f:
            f.write(command[0])
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    for name in ("OUT", "TORCH_OUT"):
        monkeypatch.setattr(B, name, str(tmp_path / os.path.basename(getattr(B, name))))
    return ran


def test_library_is_built_without_torch(compilers, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises ImportError
    assert B.build(verbose=False) == B.OUT
    assert compilers == ["nvcc"] and os.path.exists(B.OUT) and not os.path.exists(B.TORCH_OUT)
    assert "torch" in capsys.readouterr().err
    compilers.clear()
    B.build(verbose=False)  # the library is up to date
    assert compilers == []


def test_library_comes_before_its_binding(compilers):
    pytest.importorskip("torch")
    B.build(verbose=False)
    assert compilers == ["nvcc", "g++"] and os.path.exists(B.TORCH_OUT)
    B.build(verbose=False)
    assert compilers == ["nvcc", "g++"]
    os.remove(B.TORCH_OUT)
    B.build(verbose=False)
    assert compilers == ["nvcc", "g++", "g++"]
    B.build(force=True, verbose=False)
    assert compilers[3:] == ["nvcc", "g++"]
