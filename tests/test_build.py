"""The build: what is compiled again when, and for which interpreter."""
import os
import subprocess

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
