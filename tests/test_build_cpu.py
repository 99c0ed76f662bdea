"""What the library's makefile builds on machines of different kinds (make -n: nothing is compiled)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_gpt2_inference_amd", "csrc")


def _steps(*overrides):
    if not shutil.which("make"):
        pytest.skip("no make")
    r = subprocess.run(["make", "-n", "-B", "-C", CSRC, *overrides], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    return r.stdout


def test_library_and_extension(tmp_path):
    (tmp_path / "Python.h").write_text("")
    out = _steps(f"PYINC={tmp_path}", "HOST=Linux x86_64")
    assert "-shared -fPIC -o ../libkvattn.so" in out and " pycall.c" in out


@pytest.mark.parametrize("override", ["PYTHON=/no/python", "PYINC=/no/headers", "HOST=Linux aarch64", "HOST=Darwin x86_64"])
def test_library_alone_where_the_extension_cannot_be(override):
    """No interpreter, no headers of it, or another machine than the calls are laid out for: the library is built, and
    the binding has ctypes."""
    out = _steps(override)
    assert "-shared -fPIC -o ../libkvattn.so" in out and "pycall.c" not in out
