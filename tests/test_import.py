"""The package in a host without torch."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)


def test_package_imports_without_torch():
    """Hosts that pass numpy arrays need no torch: the package, its modules for them and a star import load with torch
    blocked."""
    r = _run("import sys; sys.modules['torch'] = None\n"
             "import colizig_b200 as cz\n"
             "from colizig_b200 import *\n"
             "print(cz.gpu.available(), cz.moe.Dims(256, 16, 4, 128).c().hidden, callable(cz.fp8.matmul_fp8_keyed))\n"
             "assert not hasattr(cz, 'attn')")
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["False", "256", "True"]


def test_package_has_attention_with_torch():
    r = _run("import colizig_b200 as cz; print(cz.attn.HEAD_DIMS, 'attn' in cz.__all__)")
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "(64, 128) True"
