"""Which kernels a call of the C ABI launches, and whether it reports a launch that fails, found on the host: the HIP runtime's
launch functions are replaced by a small library that records the names and fails the launch it is told to, in a process of
its own. No kernel runs, and made-up addresses are never read."""
from __future__ import annotations

import json
import os
import re
import shutil
import subprocess
import sys
import tempfile

STUB = r"""
#include <string.h>
typedef struct { unsigned x, y, z; } dim3;
static const void* key[4096]; static const char* name[4096]; static int n;
static char log_[1 << 16];
static int launched, fail_at = -1, last;
static dim3 g, b; static unsigned long sh; static void* st;
const char* stub_log(void) { return log_; }
int stub_count(void) { return n; }
const char* stub_name(int i) { return name[i]; }
void stub_reset(int k) { log_[0] = 0; launched = 0; fail_at = k; last = 0; }
void** __hipRegisterFatBinary(const void* d) { static void* h; return &h; }
void __hipUnregisterFatBinary(void** m) {}
void __hipRegisterFunction(void** m, const void* f, char* d, const char* nm, unsigned t, void* a, void* b_, void* c, void* e, int* w) {
    if (n < 4096 && strstr(nm, "mi355moe")) { key[n] = f; name[n] = nm; n++; }
}
void __hipRegisterVar(void** m, void* v, char* h, char* d, int e, unsigned long s, int c, int gl) {}
int hipLaunchKernel(const void* f, dim3 gr, dim3 bl, void** a, unsigned long s, void* q) {
    if (!gr.x || !gr.y || !gr.z) return last = 9;
    if (launched++ == fail_at) return last = 719;
    for (int i = 0; i < n; ++i)
        if (key[i] == f && strlen(log_) + strlen(name[i]) + 2 < sizeof(log_)) { strcat(log_, name[i]); strcat(log_, "\n"); return 0; }
    return last = 98;
}
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipDeviceGetAttribute(int* v, int a, int d) { *v = 256; return 0; }
int hipStreamIsCapturing(void* s, int* c) { *c = 0; return 0; }
int __hipPushCallConfiguration(dim3 gr, dim3 bl, unsigned long s, void* q) { g = gr; b = bl; sh = s; st = q; return 0; }
int __hipPopCallConfiguration(dim3* gr, dim3* bl, unsigned long* s, void** q) { *gr = g; *bl = b; *s = sh; *q = st; return 0; }
"""

CHILD = r"""
import ctypes, json, sys
sys.path.insert(0, sys.argv[2])
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
stub.stub_log.restype = ctypes.c_char_p
from mi355moe import _lib
L = _lib.lib()
P, NUL, BIG = ctypes.c_void_p(0x10000), ctypes.c_void_p(0), 1 << 44
DT = {"fp32": _lib.F32, "fp16": _lib.F16, "bf16": _lib.BF16}

def matmul(M, N, K, dt="bf16"):
    return L.mi355moe_mxfp4_matmul(P, P, M, P, P, N, K, P, DT[dt], N, P, BIG, NUL)

def moe(n, H, I, T, k, n_global=0, arranged=1):
    d = _lib.Mxfp4LayerDesc()
    d.n, d.hidden, d.intermediate, d.arranged = n, H, I, arranged
    for f in ("w13", "w13_scale", "w2", "w2_scale"):
        setattr(d, f, P)
    return L.mi355moe_mxfp4_moe_forward_ids(ctypes.byref(d), P, DT["bf16"], H, T, P, _lib.I32, P, DT["fp32"], k,
                                            P if n_global else NUL, n_global, 10.0, P, DT["bf16"], H, 0, P, BIG, NUL)

def quant(rows, K, dt="bf16"):
    return L.mi355moe_mxfp4_quant_rows(P, DT[dt], rows, K, K, P, P, NUL)

def dequant(rows, K, dt="bf16"):
    return L.mi355moe_mxfp4_dequant_rows(P, P, rows, K, P, DT[dt], NUL)

def arrange(mats, rows, K):
    return L.mi355moe_mxfp4_arrange_scales(P, mats, rows, K, P, NUL)

def forward(T, H, I, dt="bf16"):
    return L.mi355moe_gated_forward(P, DT[dt], T, H, H, P, I, 10.0, P, I, P, P, BIG, NUL)

def dx(T, H, I, dt="bf16"):
    return L.mi355moe_gated_backward(P, I, P, P, DT[dt], T, H, H, P, I, 10.0, P, NUL, P, BIG, NUL)

def dw(T, H, I, dt="bf16"):
    return L.mi355moe_gated_backward(P, I, P, P, DT[dt], T, H, H, P, I, 10.0, NUL, P, P, BIG, NUL)

stub.stub_name.restype = ctypes.c_char_p
out = [[stub.stub_name(i).decode() for i in range(stub.stub_count())]]
silent = []
for fn, args in json.load(sys.stdin):
    stub.stub_reset(-1)
    rc = globals()[fn](*args)
    assert rc == 0, (fn, args, rc)
    out.append(stub.stub_log().decode().split())
    for k in range(len(out[-1])):
        stub.stub_reset(k)
        if globals()[fn](*args) == 0:
            silent.append([fn, args, k, out[-1]])
json.dump([out, silent], sys.stdout)
"""


def _plain(mangled: str) -> str:
    """kernel<1,2,..> of a mangled name of the library's namespace."""
    m = re.match(r"_ZN8mi355moe(\d+)", mangled)
    if not m:
        return mangled
    at, size = m.end(), int(m.group(1))
    args = re.match(r"I((?:L[ib]n?\d+E|[a-z])+)E", mangled[at + size:])
    vals = re.findall(r"L[ib](\d+)E", args.group(1)) if args else []
    return mangled[at:at + size] + (f"<{','.join(vals)}>" if vals else "")


def compiler():
    return shutil.which("gcc") or shutil.which("cc") or shutil.which("clang")


def kernels():
    """The kernels that the library holds."""
    return [_plain(k) for k in _run([])[0][0]]


def launches(calls):
    """For each call (name, arguments) of the child's functions, the kernels it launches, in order."""
    return [[_plain(k) for k in names] for names in _run(calls)[0][1:]]


def silent_failures(calls):
    """The calls that report success although a launch of theirs fails: [name, arguments, which launch, the launches]."""
    return _run(calls)[1]


def _run(calls):
    from conftest import PKG_DIR
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "stub.c"), os.path.join(d, "libstub.so")
        with open(src, "w") as f:
            f.write(STUB)
        subprocess.run([compiler(), "-shared", "-fPIC", "-w", "-o", so, src], check=True, timeout=60)
        r = subprocess.run([sys.executable, "-c", CHILD, so, PKG_DIR], input=json.dumps(calls), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-1500:]
    return json.loads(r.stdout)
