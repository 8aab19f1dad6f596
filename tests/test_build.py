"""What build.py builds again, and what it builds without torch: with a compiler that only touches its output."""
import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "semantic-ai_b200" / "build.py"


@pytest.fixture
def builder(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("svl_build_under_test", SOURCE)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.OUT, b.LIB, b.TORCH_OPS = tmp_path / "out", tmp_path / "lib.so", tmp_path / "_torch_ops.so"
    b.made, b.fails = [], set()

    def compiler(cmd, **_):
        target = Path(cmd[cmd.index("-o") + 1])
        if target.name in b.fails:
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        target.touch()
        b.made.append(target.name)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b.subprocess, "run", compiler)
    return b


def test_nothing_is_built_twice(builder):
    assert builder.build() == builder.LIB
    assert {"lib.so", "_torch_ops.so", "rules.o"} <= set(builder.made)
    builder.made.clear()
    builder.build()
    assert builder.made == []


def test_the_binding_follows_torch(builder, monkeypatch):
    """Another torch, or a binding whose build nothing is known of: built again."""
    import torch
    builder.build()
    builder.made.clear()
    monkeypatch.setattr(torch, "__version__", "0.0.another")
    builder.build()
    assert builder.made == ["_torch_ops.so"]
    builder.made.clear()
    for f in builder.OUT.glob("*.stamp"):
        f.unlink()
    builder.build()
    assert builder.made == ["_torch_ops.so"]


def test_the_library_without_torch(builder, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert builder.build() == builder.LIB
    assert "lib.so" in builder.made and "_torch_ops.so" not in builder.made
    assert "torch" in capsys.readouterr().err


def test_a_failed_binding_leaves_the_library(builder):
    builder.fails.add("_torch_ops.so")
    with pytest.raises(RuntimeError, match="_torch_ops.so"):
        builder.build()
    assert builder.LIB.exists()
    builder.fails.clear()
    builder.made.clear()
    builder.build()
    assert builder.made == ["_torch_ops.so"]
