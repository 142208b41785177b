"""Sizes of the calls around a layer's experts (tokens by expert, the dense product, the norms), with the kernels that each is
there for. tests/test_block_paths.py holds the kernels to that on the host; tests/test_gpu_block_paths.py runs the calls."""
from __future__ import annotations

import launches

CHILD = r"""
import ctypes, json, sys
sys.path.insert(0, sys.argv[2])
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
stub.stub_log.restype = ctypes.c_char_p
from mi355moe import _lib
L = _lib.lib()
P, NUL, BIG = ctypes.c_void_p(0x10000), ctypes.c_void_p(0), 1 << 44
DT = {"fp32": _lib.F32, "fp16": _lib.F16, "bf16": _lib.BF16}

def sort(T, k, n, wide=0):
    return L.mi355moe_sort_tokens(P, _lib.I64 if wide else _lib.I32, T, k, NUL, 0, n, P, P, P, P, BIG, NUL)

def to(T, k, H, dt="bf16"):
    return L.mi355moe_rows_to_experts(P, DT[dt], T, H, H, P, k, P, NUL)

def back(T, k, H, dt="bf16"):
    return L.mi355moe_rows_from_experts(P, DT[dt], T, H, P, k, P, _lib.F32, P, H, P, H, NUL)

def back_grad(T, k, H, dt="bf16"):
    return L.mi355moe_rows_from_experts_backward(P, DT[dt], T, H, H, P, k, P, _lib.F32, P, P, P, NUL)

def linear(M, K, N, dt="bf16"):
    return L.mi355moe_linear_forward(P, DT[dt], M, K, K, P, N, K, P, _lib.F32, 2, P, N, P, N, P, P, BIG, NUL)

def dx(M, K, N, dt="bf16", act=0):
    return L.mi355moe_linear_backward(P, N, P, P, DT[dt], M, K, K, P, N, K, act, P, NUL, NUL, _lib.F32, P, BIG, NUL)

def dw(M, K, N, dt="bf16", act=0):
    return L.mi355moe_linear_backward(P, N, P, P, DT[dt], M, K, K, P, N, K, act, NUL, P, NUL, _lib.F32, P, BIG, NUL)

def grads(M, K, N, dt="bf16", act=2):
    return L.mi355moe_linear_backward(P, N, P, P, DT[dt], M, K, K, P, N, K, act, P, P, P, _lib.F32, P, BIG, NUL)

def norm(R, H, dt="bf16"):
    return L.mi355moe_norm_forward(P, DT[dt], R, H, H, P, H, P, P, _lib.F32, P, _lib.F32, 1, 1e-5, 1.0, 1.0, P, P, P, NUL)

def norm_grad(R, H, dt="bf16", weights=1):
    w = P if weights else NUL
    return L.mi355moe_norm_backward(P, H, P, H, P, DT[dt], R, H, H, P, H, P, P, _lib.F32, P, _lib.F32, 1, 1.0, 1.0, P, P, P, w, w, w, P, BIG, NUL)

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


def run(calls):
    """([the library's kernels, the kernels of each call], the calls that report success although a launch of theirs fails)."""
    kept, launches.CHILD = launches.CHILD, CHILD
    try:
        out, silent = launches._run(calls)
    finally:
        launches.CHILD = kept
    return [[launches._plain(k) for k in names] for names in out], silent


def _tiles(p, q, shape):
    return f"linear_kernel<2,{p},{q},{shape}>"


S64, DEEP, WIDE, BIG = "64,64,2,2,4", "128,128,2,4,4", "256,128,2,4,3", "256,256,2,4,2"
JOIN, PAD = "linear_join_kernel<2>", "linear_pad_kernel"

# M, K, N, the kernels of the forward pass (bf16; fp16's are the same ones)
LINEAR = [
    (1, 136, 72, ["linear_few_kernel<2>"]),
    (33, 1027, 70, ["linear_few_kernel<2>"]),
    (300, 264, 776, [_tiles(0, 0, S64)]),
    (900, 131, 777, ["linear_any_kernel<2>"]),
    (4200, 37, 70, ["linear_any_kernel<2>"]),
    (130, 4099, 1032, ["linear_any_kernel<2>", JOIN]),
    (130, 4104, 1032, [_tiles(0, 0, S64), JOIN]),
    (1030, 4104, 2056, [_tiles(0, 0, DEEP)]),
    (1030, 4099, 1032, [PAD, _tiles(0, 0, DEEP), JOIN]),
    (2100, 1096, 2056, [_tiles(0, 0, WIDE)]),
    (2570, 1096, 5128, [_tiles(0, 0, BIG)]),
]
# the products of the gradients (without an activation): dx from dout [M][N] and w [N][K], then dw from dout and x [M][K]
DX = [
    (130, 264, 136, [_tiles(1, 0, S64)]),
    (130, 267, 133, ["linear_dz_kernel<2>", PAD, _tiles(1, 0, S64)]),
    (130, 1032, 4104, [_tiles(1, 0, S64), JOIN]),
    (1030, 2056, 4104, [_tiles(1, 0, DEEP)]),
    (1030, 1032, 4104, [_tiles(1, 0, DEEP), JOIN]),
    (2100, 2056, 1096, [_tiles(1, 0, WIDE)]),
    (2570, 5128, 1096, [_tiles(1, 0, BIG)]),
]
DW = [
    (130, 264, 136, [_tiles(1, 1, S64)]),
    (133, 267, 131, ["linear_dz_kernel<2>", PAD, _tiles(1, 1, S64)]),
    (4103, 264, 136, [_tiles(1, 1, S64), JOIN]),
    (4099, 2056, 1032, [_tiles(1, 1, DEEP)]),
    (4099, 1032, 1032, [_tiles(1, 1, DEEP), JOIN]),
    (1097, 2056, 2104, [_tiles(1, 1, WIDE)]),
    (1099, 5128, 2568, [_tiles(1, 1, BIG)]),
]

# rows, H, the kernels of the forward pass, of the gradient (weights and the gate's among it)
NORM = [
    (9, 512, ["norm_kernel<2,0,1,0>"], ["norm_grad_kernel<2,0>", "norm_join_kernel"]),
    (9, 520, ["norm_kernel<2,1,1,0>"], ["norm_grad_kernel<2,1>", "norm_join_kernel"]),
    (4098, 8190, ["norm_kernel<2,1,1,1>"], ["norm_grad_kernel<2,1>", "norm_join_kernel"]),
    (5, 8200, ["norm_kernel<2,1,2,0>"], ["norm_grad_long_kernel<2>", "norm_join_kernel"]),
]

# tokens, topk, H, the kernels of the way out, of the way back, of its gradient
ROWS = [
    (40, 6, 72, ["rows_scatter_kernel<2,0>"], ["rows_gather_kernel<2,0,0>"], ["rows_grad_kernel<2,0>"]),
    (40, 6, 520, ["rows_scatter_kernel<2,1>"], ["rows_gather_kernel<2,1,0>"], ["rows_grad_kernel<2,0>"]),
    (4100, 8, 1035, ["rows_scatter_kernel<2,1>"], ["rows_gather_kernel<2,1,1>"], ["rows_grad_kernel<2,1>"]),
]
# tokens, topk, experts, the kernels
SORT = [
    (512, 8, 288, ["sort_place_kernel"]),
    (513, 8, 288, ["sort_count_kernel", "sort_place_kernel"]),
]
