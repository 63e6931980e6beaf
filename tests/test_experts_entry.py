"""CPU suite: entry points of the operators around a router whose host side can be seen without a GPU."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def call(body):
    """Runs `body` in a process of its own that sees no GPU, so that nothing is ever launched on the made-up addresses; what it printed."""
    script = "import ctypes as C\nfrom nacho_b200 import _capi\nfrom nacho_b200._capi import DenseStruct, Fp8Struct, lib\n" + body
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    return r.stdout.strip()


def test_a_product_without_experts_returns():
    """Rows of no expert are zeros, also where there are no experts at all: without a GPU the call fails, it does not end the process."""
    assert call("""
a, w, y = Fp8Struct(1, 5, 256, 0, 4096, 8192), Fp8Struct(0, 16, 256, 1, 12288, 16384), DenseStruct(5, 16, 16, 0, 20480)
print(lib.nb200_fp8_product(C.byref(a), C.byref(w), C.c_void_p(24576), C.byref(y), None) == _capi.E_CUDA)
print(lib.nb200_fp8_product(C.byref(a), C.byref(w), None, C.byref(y), None) == _capi.E_BADARG)
""").split() == ["True", "True"]
