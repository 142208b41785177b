"""A kernel launch that fails is reported by the call that made it, whichever of its launches it is. The HIP runtime's launch
functions are replaced by a small library that fails the k-th launch, in a process of its own; no GPU needed, and no kernel
runs (made-up addresses are never read)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import textwrap

import pytest

STUB = r"""
typedef struct { unsigned x, y, z; } dim3;
static int launches, fail_at = -1, last;
static dim3 g, b; static unsigned long sh; static void* st;
void stub_reset(int k) { launches = 0; fail_at = k; last = 0; }
int stub_launches(void) { return launches; }
int hipLaunchKernel(const void* f, dim3 gr, dim3 bl, void** a, unsigned long s, void* q) {
    if (gr.x == 0 || gr.y == 0 || gr.z == 0) return last = 9;
    if (launches++ == fail_at) return last = 719;
    return 0;
}
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipPeekAtLastError(void) { return last; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipDeviceGetAttribute(int* v, int a, int d) { *v = 256; return 0; }
int hipStreamIsCapturing(void* s, int* c) { *c = 0; return 0; }
int __hipPushCallConfiguration(dim3 gr, dim3 bl, unsigned long s, void* q) { g = gr; b = bl; sh = s; st = q; return 0; }
int __hipPopCallConfiguration(dim3* gr, dim3* bl, unsigned long* s, void** q) { *gr = g; *bl = b; *s = sh; *q = st; return 0; }
"""

CHILD = r"""
import ctypes, sys
sys.path.insert(0, sys.argv[3])
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from mi355moe import _lib
L = _lib.lib()
P, NUL, BIG = ctypes.c_void_p(0x10000), ctypes.c_void_p(0), 1 << 40
F32, F16, BF16, I32 = _lib.F32, _lib.F16, _lib.BF16, _lib.I32

def matmul(M, N, K):
    return lambda: L.mi355moe_mxfp4_matmul(P, P, M, P, P, N, K, P, BF16, N, P, BIG, NUL)

def moe(n, H, I, T, k):
    d = _lib.Mxfp4LayerDesc()
    d.n, d.hidden, d.intermediate, d.arranged = n, H, I, 1
    for f in ("w13", "w13_scale", "w2", "w2_scale"):
        setattr(d, f, P)
    return lambda: L.mi355moe_mxfp4_moe_forward_ids(ctypes.byref(d), P, BF16, H, T, P, I32, P, F32, k, NUL, 0, 10.0, P, BF16, H, 0, P, BIG, NUL)

def fwd(T, H, I, dt=BF16):
    return lambda: L.mi355moe_gated_forward(P, dt, T, H, H, P, I, 10.0, P, I, P, P, BIG, NUL)

def bwd(T, H, I, dt=BF16):
    return lambda: L.mi355moe_gated_backward(P, I, P, P, dt, T, H, H, P, I, 10.0, P, P, P, BIG, NUL)

calls = {
    "quant": (1, lambda: L.mi355moe_mxfp4_quant_rows(P, BF16, 9, 64, 64, P, P, NUL)),
    "dequant": (1, lambda: L.mi355moe_mxfp4_dequant_rows(P, P, 9, 64, P, BF16, NUL)),
    "arrange": (1, lambda: L.mi355moe_mxfp4_arrange_scales(P, 2, 5, 96, P, NUL)),
    "product, few rows": (1, matmul(1, 4096, 4096)),
    "product, tiles": (1, matmul(1024, 4096, 4096)),
    "product, largest tiles": (2, matmul(8192, 4096, 4096)),
    "product, parts": (2, matmul(128, 512, 32768)),
    "product, arranged and in parts": (3, matmul(128, 512, 32768 + 32)),
    "experts, few pairs": (2, moe(288, 4096, 1024, 1, 8)),
    "experts, few rows": (4, moe(288, 4096, 1024, 64, 8)),
    "experts, tiles": (4, moe(288, 4096, 1024, 2047, 8)),
    "experts, wide tiles": (4, moe(36, 4096, 1024, 2047, 8)),
    "gated, few rows": (1, fwd(1, 4096, 1024)),
    "gated, parts": (2, fwd(200, 4096, 1024)),
    "gated, tiles": (1, fwd(1791, 4096, 1024)),
    "gradients": (3, bwd(1791, 4096, 1024)),
    "gradients, fp16": (4, bwd(1791, 4096, 1024, F16)),
    "gradients, dx in parts": (4, bwd(130, 264, 2056)),
    "gradients, dw13 in parts": (4, bwd(8192, 128, 64)),
}
for name, (least, call) in calls.items():
    stub.stub_reset(-1)
    assert call() == 0, name
    n = stub.stub_launches()
    assert n >= least, (name, n)
    for k in range(n):
        stub.stub_reset(k)
        assert call() != 0, "%s: launch %d of %d failed and the call reported success" % (name, k + 1, n)
        stub.stub_reset(-1)
        assert call() == 0, name
print("all reported")
"""


def test_failed_launches_are_reported(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc") or shutil.which("clang")
    if not cc:
        pytest.skip("no C compiler")
    from conftest import PKG_DIR
    (tmp_path / "stub.c").write_text(STUB)
    so = tmp_path / "libstub.so"
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(so), str(tmp_path / "stub.c")], check=True, timeout=60)
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(CHILD), str(so), os.path.dirname(PKG_DIR), PKG_DIR], capture_output=True,
                       text=True, timeout=240)
    assert r.returncode == 0 and "all reported" in r.stdout, r.stdout[-500:] + r.stderr[-1500:]
