"""The extension that takes the small calls: where it cannot be built or used, the library is built and used without it."""
import os
import subprocess
import warnings

import pytest
import torch

from trellis_b200 import _lib, experts


@pytest.fixture
def unloaded(monkeypatch):
    _lib.lib()
    monkeypatch.setattr(_lib, "_short", None)


def refused_as_ever():
    for call in (lambda: experts.route(torch.zeros(2, 4), 2), lambda: experts.quantize_experts(torch.zeros(2, 4, 32))):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_it_is_loaded_for_what_runs(unloaded):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        module = _lib.short()
    assert module and module is _lib.short() and module.built_for[0] == _lib.ABI_VERSION and torch.__version__.startswith(module.built_for[1])


def test_without_it(unloaded, monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "SHORT_PATH", str(tmp_path / "tcq_torch.so"))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert _lib.short() is False
    refused_as_ever()


def test_one_that_cannot_be_loaded(unloaded, monkeypatch, tmp_path):
    """A warning, once, and the calls go the other way."""
    (tmp_path / "tcq_torch.so").write_bytes(b"of another machine")
    monkeypatch.setattr(_lib, "SHORT_PATH", str(tmp_path / "tcq_torch.so"))
    with pytest.warns(RuntimeWarning, match="ctypes"):
        assert _lib.short() is False
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert _lib.short() is False
        refused_as_ever()


@pytest.mark.parametrize("what", ["abi", "torch"])
def test_one_that_was_built_for_something_else(unloaded, monkeypatch, what):
    if what == "abi":
        monkeypatch.setattr(_lib, "ABI_VERSION", _lib.ABI_VERSION + 1)
    else:
        monkeypatch.setattr(torch, "__version__", "1.0.0+cu1")
    with pytest.warns(RuntimeWarning, match="built for"):
        assert _lib.short() is False
    refused_as_ever()


def test_the_library_is_built_without_it(monkeypatch):
    def run(broken):
        made = []

        def make(cmd, **_):
            made.extend(c for c in cmd if c.endswith(".so"))
            if broken in cmd:
                raise subprocess.CalledProcessError(2, cmd)
        monkeypatch.setattr(subprocess, "check_call", make)
        return _lib.build(), made
    assert run("nothing") == (_lib.LIB_PATH, ["libtcq_b200.so", "tcq_torch.so"])
    with pytest.warns(RuntimeWarning, match="not built"):
        assert run("tcq_torch.so") == (_lib.LIB_PATH, ["libtcq_b200.so", "tcq_torch.so"])
    with pytest.raises(subprocess.CalledProcessError):
        run("libtcq_b200.so")


def test_make_builds_both():
    csrc = os.path.dirname(_lib.LIB_PATH)
    plan = subprocess.run(["make", "-n", "-B", "-C", csrc], capture_output=True, text=True, check=True).stdout
    assert "libtcq_b200.so" in plan and "tcq_torch.cpp" in plan


def test_what_is_no_routing():
    for bad in ((1, 2, 3), [None] * 5, None, torch.zeros(5)):
        with pytest.raises(ValueError):
            experts.combine(torch.zeros(2, 4), bad)
