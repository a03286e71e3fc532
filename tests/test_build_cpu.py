"""What build() compiles, with its compiler calls recorded instead of run."""

import os
import subprocess

import pytest

from megamoe import _build


class Recorder:
    def __init__(self, monkeypatch):
        self.commands = []
        monkeypatch.setattr(_build, "_run", self)

    def __call__(self, cmd, verbose):
        self.commands.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    def outputs(self):
        return sorted(os.path.basename(c[c.index("-o") + 1]) for c in self.commands)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A built tree of its own: build() finds nothing to do in it."""
    monkeypatch.setattr(_build, "OUTPUT", str(tmp_path / "libmegamoe.so"))
    monkeypatch.setattr(_build, "TORCH_OUTPUT", str(tmp_path / "_dense.so"))
    monkeypatch.setattr(_build, "OBJDIR", str(tmp_path / "_build"))
    run = Recorder(monkeypatch)
    _build.build()
    assert "libmegamoe.so" in run.outputs() and "_dense.so" in run.outputs()
    run.commands.clear()
    _build.build()
    assert run.commands == []
    return run


def test_a_newer_binding_source_costs_one_compilation(tree, monkeypatch):
    old = os.path.getmtime(os.path.join(_build.CSRC, _build.TORCH_SOURCE)) - 10
    os.utime(_build.TORCH_OUTPUT, (old, old))
    _build.build()
    assert tree.outputs() == ["_dense.so"]


def test_a_newer_kernel_source_builds_the_library(tree):
    old = max(os.path.getmtime(os.path.join(_build.CSRC, f)) for f in _build.SOURCES) - 10
    os.utime(_build.OUTPUT, (old, old))
    _build.build()
    assert "libmegamoe.so" in tree.outputs() and "mm_norm.o" in tree.outputs()


def test_force_builds_everything(tree):
    _build.build(force=True)
    assert tree.outputs() == sorted(["libmegamoe.so", "_dense.so"] + [s.replace(".cu", ".o") for s in _build.SOURCES])


@pytest.mark.parametrize("what", ["torch", "python"])
def test_the_binding_is_built_again_for_another_torch_or_python(tree, monkeypatch, what):
    import sysconfig

    import torch

    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    else:
        real = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda n: "cpython-399" if n == "SOABI" else real(n))
    _build.build()
    assert tree.outputs() == ["_dense.so"]
    tree.commands.clear()
    _build.build()
    assert tree.commands == []


def test_a_host_without_the_headers_still_builds_the_library(tree, monkeypatch, tmp_path, capsys):
    """Python.h missing: the library (the MoE chain) is built, the binding is named as left out,
    and one compiled for other headers does not stay behind to be loaded."""
    import sysconfig

    real = sysconfig.get_paths
    monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: dict(real(*a, **k), include=str(tmp_path / "none")))
    assert _build.build(force=True) == _build.OUTPUT
    assert "libmegamoe.so" in tree.outputs() and "_dense.so" not in tree.outputs()
    assert not os.path.exists(_build.TORCH_OUTPUT)
    err = capsys.readouterr().err
    assert "_dense.so" in err and "Python.h" in err


def test_a_compiler_error_is_an_error(tree, monkeypatch):
    monkeypatch.setattr(_build, "_run", lambda cmd, verbose: subprocess.CompletedProcess(cmd, 1, "", "no"))
    os.remove(_build.TORCH_OUTPUT)
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        _build.build()


def test_calls_without_the_binding_say_what_is_missing(monkeypatch):
    import sys

    import megamoe
    from megamoe import dense

    monkeypatch.setattr(dense, "_dense", None)
    monkeypatch.setitem(sys.modules, "megamoe._dense", None)
    monkeypatch.delattr(megamoe, "_dense", raising=False)
    with pytest.raises(RuntimeError, match="_dense.so does not load"):
        megamoe.quantize_int8(None)
