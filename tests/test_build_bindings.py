"""neuroflow_cpp needs pybind11 and the library alone: it is built where torch is not installed."""
import sys

import pytest

from neuroflow_amd import build as nb


@pytest.fixture
def built(monkeypatch):
    names = []
    monkeypatch.setattr(nb, "_build_binding", lambda name, flags, verbose: names.append(name) or nb.LIB_DIR / name)
    return names


def test_without_torch(built, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)          # import torch raises ImportError
    assert nb.build_bindings().name == "neuroflow_cpp"
    assert built == ["neuroflow_cpp"]
    assert "block_ops" in capsys.readouterr().out


def test_with_torch(built):
    nb.build_bindings(verbose=False)
    assert sorted(built) == ["block_ops", "neuroflow_cpp"]


def test_a_torch_module_that_does_not_build_leaves_the_other(monkeypatch):
    names = []

    def fails(name, flags, verbose):
        if name == "block_ops":
            raise RuntimeError("bindings build failed")
        names.append(name)
    monkeypatch.setattr(nb, "_build_binding", fails)
    with pytest.raises(RuntimeError):
        nb.build_bindings()
    assert names == ["neuroflow_cpp"]
