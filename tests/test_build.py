"""The build: what is compiled again when, and for which interpreter."""
import os
import subprocess
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ayolov2_amd", "csrc")


def _would_run(*args):
    return subprocess.run(["make", "-n", "-C", CSRC, *args], capture_output=True, text=True, check=True).stdout


def test_changed_flags_compile_everything_again():
    """the flags stand in the Makefile, and objects of other flags must not stay"""
    out = _would_run("-W", "Makefile")
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    assert len(sources) >= 10
    for f in sources:
        assert f"-c {f} -o _build/{f[:-4]}.o" in out and "-packed-fp32-ops" in out
    assert "host.cpp -o ../_host.so" in out


def test_build_is_for_the_interpreter_that_runs_it(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "check_call", lambda args: calls.append(args))
    entry.build()
    assert calls[0][0] == "make" and f"PYTHON={sys.executable}" in calls[0] and "-B" in calls[0]
    out = _would_run("-W", "host.cpp", f"PYTHON={sys.executable}")
    import torch
    assert f"-isystem {os.path.dirname(torch.__file__)}/include" in out


def test_a_helper_of_another_build_is_refused():
    import torch

    from ayolov2_amd import _lib
    mod = _lib.host()
    assert mod.built_for_torch == ".".join(torch.__version__.split(".")[:3]).split("+")[0].split("a")[0]
    for py, tv in (("3.99.1", mod.built_for_torch), (mod.built_for_python, "1.0.0")):
        with pytest.raises(_lib.AyoloError, match="build it again"):
            _lib._check_host(types.SimpleNamespace(built_for_python=py, built_for_torch=tv))
    with pytest.raises(_lib.AyoloError, match="build it again"):
        _lib._check_host(types.SimpleNamespace())          # built before it said for what
    _lib._check_host(mod)
