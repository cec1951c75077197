"""What build.py compiles, with every compiler call recorded instead of run."""
from __future__ import annotations

import importlib.util
import os
import sys

import pytest

from conftest import ROOT


class NoTorch:
    def find_spec(self, name, path=None, target=None):
        if name == "torch" or name.startswith("torch."):
            raise ModuleNotFoundError(f"No module named {name!r}", name=name)


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with outputs in a folder of the test; `ran` holds the sources of the g++ calls."""
    spec = importlib.util.spec_from_file_location("_builder", os.path.join(ROOT, "flash_attn_metal_cpp_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    lib = tmp_path / "libfa_b200.so"
    lib.touch()
    b.LIB, b.EXT, b.EXT_PAGED, b.OBJDIR = (str(tmp_path / n) for n in ("libfa_b200.so", "module.so", "paged.so", "_build"))
    b.ran = []

    def run(cmd):
        b.ran.append(next(os.path.basename(c) for c in cmd if c.endswith(".cpp")))
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(b, "NVCC", sys.executable)
    monkeypatch.setattr(b, "_compile", lambda src, force: str(lib))
    monkeypatch.setattr(b, "_run", run)
    return b


@pytest.fixture
def no_torch(monkeypatch):
    for n in [n for n in sys.modules if n == "torch" or n.startswith("torch.")]:
        monkeypatch.delitem(sys.modules, n)
    monkeypatch.setattr(sys, "meta_path", [NoTorch(), *sys.meta_path])


def test_both_extensions(builder):
    builder.build()
    assert sorted(builder.ran) == ["bindings.cpp", "bindings_paged.cpp"]


def test_the_module_is_built_without_torch(builder, no_torch, capsys):
    builder.build()
    assert builder.ran == ["bindings.cpp"]
    assert "paged" in capsys.readouterr().err


def test_a_torch_without_cuda_counts_as_none(builder, monkeypatch):
    import torch

    monkeypatch.setattr(torch.version, "cuda", None)
    builder.build()
    assert builder.ran == ["bindings.cpp"]


def test_another_torch_rebuilds_what_uses_it(builder, monkeypatch):
    import torch

    builder.build()
    builder.ran.clear()
    builder.build()
    assert builder.ran == []
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    builder.build()
    assert builder.ran == ["bindings_paged.cpp"]
    builder.build()
    assert builder.ran == ["bindings_paged.cpp"]
