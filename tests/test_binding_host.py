"""The native binding of the calls between logits and an update where it cannot
be used (CPU only): the general path takes the calls, with a warning, and the
build neither needs torch nor keeps a binding of another one."""
import subprocess
import sys
import types
import warnings

import pytest

import kernix_b200 as kx
from kernix_b200 import _build


@pytest.fixture
def anew(monkeypatch):
    """_native as a fresh process finds it."""
    kx._native.cache_clear()
    yield monkeypatch
    kx._native.cache_clear()


def replaced(monkeypatch, module):
    monkeypatch.setitem(sys.modules, "kernix_b200._kx_torch", module)
    monkeypatch.delattr(kx, "_kx_torch", raising=False)
    if module is not None:
        monkeypatch.setattr(kx, "_kx_torch", module, raising=False)


def check_general(match):
    with pytest.warns(RuntimeWarning, match=match):
        native = kx._native()
    assert native.token_log_probs(1, 2) is native.token_log_probs_backward() is native.grad_norm(3) is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert kx._native() is native       # once


def test_no_binding(anew):
    replaced(anew, None)                    # importing it raises ImportError
    check_general("no native binding")


def test_a_binding_for_another_torch(anew):
    other = types.ModuleType("kernix_b200._kx_torch")
    other.torch = "1.0.0"
    other.bind = lambda *_: pytest.fail("used")
    replaced(anew, other)
    check_general("built for torch 1.0.0")


def test_the_binding_of_this_torch(anew):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        native = kx._native()
    assert native.__name__ == "kernix_b200._kx_torch"


def test_calls_without_the_binding_refuse_as_ever(anew):
    import torch
    replaced(anew, None)
    with pytest.warns(RuntimeWarning), pytest.raises(kx.NoDevice):
        kx.token_log_probs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(kx.NoDevice):
        kx.grad_norm([torch.zeros(3)])


def test_the_build_leaves_the_binding_out_without_torch(monkeypatch, capfd):
    monkeypatch.setattr(_build.importlib.util, "find_spec", lambda name: None)
    monkeypatch.setattr(subprocess, "run", lambda *a, **k: pytest.fail("compiled"))
    _build._binding(force=True, verbose=False)
    assert "left out" in capfd.readouterr().err


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """Its version decides, not the files' times; a build that fails leaves
    nothing behind that passes for one."""
    torch = tmp_path / "torch"
    (torch / "include" / "ATen").mkdir(parents=True)
    (torch / "include" / "ATen" / "ATen.h").touch()
    (torch / "version.py").write_text("__version__ = '1'")
    runs = []

    def run(cmd, check):
        runs.append(cmd)
        if not fail:
            open(cmd[cmd.index("-o") + 1], "w").close()
        else:
            raise subprocess.CalledProcessError(1, cmd)

    monkeypatch.setattr(_build.importlib.util, "find_spec",
                        lambda name: types.SimpleNamespace(submodule_search_locations=[str(torch)]))
    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(_build, "PKG", tmp_path)
    monkeypatch.setattr(_build, "OBJ", tmp_path)
    monkeypatch.setattr(_build, "BINDING", tmp_path / "_kx_torch.x.so")
    fail = False
    _build._binding(False, False)
    _build._binding(False, False)
    assert len(runs) == 1
    (torch / "version.py").write_text("__version__ = '2'")
    fail = True
    with pytest.raises(subprocess.CalledProcessError):
        _build._binding(False, False)
    fail = False
    _build._binding(False, False)
    _build._binding(False, False)
    assert len(runs) == 3 and all(str(torch / "include") in c for c in runs)
