"""What the library's build asks of a host."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "colizig_b200", "csrc")


def _would_run(*targets):
    r = subprocess.run(["make", "-n", "-B", "-C", CSRC, "PYTHON=no-such-python", *targets], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stderr
    return r.stdout, r.stderr


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_library_builds_without_python_and_torch():
    """A host of the C interface (the reference's is Zig) runs plain make: no interpreter, no torch headers."""
    out, err = _would_run()
    assert "libcolizig_cuda.so" in out
    assert "attn_binding" not in out and "no-such-python" not in out + err


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_binding_is_a_target_of_its_own():
    assert "attn_binding.cpp" in _would_run("binding")[0]
