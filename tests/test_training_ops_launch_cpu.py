"""A kernel that cannot be launched is an error of the call, whichever of the call's launches it is.

A child process loads the library behind a stand-in for the CUDA runtime's launches, which launches nothing and fails where it
is told to.  No kernel runs, so the pointers are stand-ins too."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

SHIM = r"""
#include <stddef.h>
static int count, fail_at = -1, last;
void shim_arm(int at) { count = 0; fail_at = at; last = 0; }
int shim_count(void) { return count; }
static int launch(void) { return count++ == fail_at ? (last = 98) : 0; }
int cudaLaunchKernel(const void* f, ...) { return launch(); }
int cudaLaunchKernelExC(const void* c, const void* f, void** a) { return launch(); }
unsigned __cudaPushCallConfiguration(void) { return 0; }
int __cudaPopCallConfiguration(void* g, void* b, size_t* m, void** s) { *m = 0; *s = 0; return 0; }
int cudaGetLastError(void) { int e = last; last = 0; return e; }
int cudaPeekAtLastError(void) { return last; }
int cudaGetDevice(int* d) { *d = 0; return 0; }
int cudaDeviceGetAttribute(int* v, int a, int d) { *v = 148; return 0; }
int cudaGetSymbolAddress(void** p, const void* s) { *p = (void*)4096; return 0; }
"""

CHILD = r"""
import ctypes as C, sys
sys.path.insert(0, sys.argv[1])
from gsa_b200 import _lib

lib = _lib.lib()
shim = C.CDLL(None)
p, big = C.c_void_p(1 << 20), 1 << 40


def calls(dtype, rows, d):
    c_ld, s_ld = (d + 15) // 16 * 16, (d + 31) // 32
    back = (p, d, None, 0, p, p, c_ld, p, s_ld, p, p, d, None, 0)
    e = d // 2 * 2
    if e <= 1024:
        side = C.byref(_lib.RotarySide(1 << 20, 1 << 21, 2, 2 * d * rows, 2 * d, d, 2 * d * rows, 2 * d, d))
        yield "rotary", lambda: lib.gsa_rotary(dtype, 1, rows, e, e, side, None, p, rows, 1, p, None, None, 0, 0, 0, 1.0, 0, 0, None)
    yield "pack", lambda: lib.gsa_pack_e4m3(dtype, rows, d, p, d, p, c_ld, p, s_ld, None)
    yield "unpack", lambda: lib.gsa_unpack_e4m3(dtype, rows, d, p, c_ld, p, s_ld, p, d, None)
    yield "silu", lambda: lib.gsa_silu_mul_pack(dtype, rows, d, p, 2 * d, p, d, p, c_ld, p, s_ld, None)
    yield "silu backward", lambda: lib.gsa_silu_mul_packed_backward(dtype, rows, d, p, d, p, c_ld, p, s_ld, p, 2 * d, None, 0, None)
    yield "norm", lambda: lib.gsa_add_rmsnorm_pack(dtype, rows, d, p, d, None, 0, p, 1e-5, None, 0, p, d, p, c_ld, p, s_ld, p, None)
    yield "norm backward", lambda: lib.gsa_rmsnorm_packed_backward(dtype, rows, d, *back, None, None, 0, None)
    yield "norm backward, dw", lambda: lib.gsa_rmsnorm_packed_backward(dtype, rows, d, *back, p, p, big, None)
    yield "loss", lambda: lib.gsa_next_token_loss(dtype, 1, rows, d, p, d * rows, d, p, rows, 1, -100, p, p, d * rows, d, p, big, None)
    yield "scale", lambda: lib.gsa_scale(dtype, d, p, p, None)


lost = []
for dtype in (_lib.DTYPE_F32, _lib.DTYPE_BF16):
    for rows, d in ((3, 64), (3, 33), (3, 2048), (3, 12000), (3, 20000), (5000, 33)):
        for name, call in calls(dtype, rows, d):
            shim.shim_arm(-1)
            assert call() == 0, (name, rows, d)
            n = shim.shim_count()
            assert n > 0, (name, rows, d)
            for at in range(n):
                shim.shim_arm(at)
                if call() == 0:
                    lost.append((name, dtype, rows, d, f"launch {at + 1} of {n}"))
print("\n".join(map(str, lost)))
sys.exit(len(lost) > 0)
"""


def test_every_failed_launch_is_reported(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("needs a C compiler")
    (tmp_path / "shim.c").write_text(SHIM)
    shim = tmp_path / "shim.so"
    subprocess.run([gcc, "-shared", "-fPIC", "-w", "-fno-builtin", str(tmp_path / "shim.c"), "-o", str(shim)], check=True)
    (tmp_path / "child.py").write_text(CHILD)
    package = Path(__file__).resolve().parent.parent / "gated-sparse-attention_b200"
    r = subprocess.run([sys.executable, str(tmp_path / "child.py"), str(package)], env={**os.environ, "LD_PRELOAD": str(shim)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
