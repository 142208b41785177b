"""Microscaled 4-bit floats (OCP MXFP4): e2m1 values with one power-of-two scale (e8m0) per 32, multiplied by gfx950's
scaled matrix instructions. No counterpart in the reference, whose 4-bit experts are EXL3's.

A row of K values is uint8 [ceil(K / 2)] codes (value 2i in the low four bits of byte i) and uint8 [ceil(K / 32)] scale
codes (2^(code - 127); 255 = NaN), the layout of MXFP4 checkpoints.

  quant_rows / dequant_rows   rows of fp32, fp16 or bf16 to codes and scales, and back
  matmul                      A W^T of two MXFP4 matrices (the contraction contiguous in both)
  Mxfp4Experts                one layer's experts: w13 [n, 2I, H/2] (gate rows, then up rows), w2 [n, H, I/2], their scales
  moe_forward_ids             routed output from router ids and weights, activations quantised per block of 32
  fused_experts_mxfp4         the functional form apply(hidden, w13, w2, topk_weights, topk_ids, scales)

Nothing here has a gradient. Codes carry none; the routed output of an x or topk_weights that needs one raises in the backward
pass, and an `out` that autograd would lose track of is refused.

Every call runs on the current stream of its tensors' device. Scratch comes from torch's caching allocator call by call
(a captured call's from its graph's own pool), so calls on several streams, and graphs replayed side by side, share none.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _addr, _need_cuda, _no_tangents, _on_device, _raw_stream, ids_dtype_code, weight_dtype_code

BLOCK = 32
SCALE_NAN = 255


def _codes(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.uint8:
        raise ValueError(f"{name} must be torch.uint8 (MXFP4 codes, scale codes), got {t.dtype}")
    return t


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def _rows(x: torch.Tensor, name: str = "x") -> torch.Tensor:
    """x as rows that do not overlap, with unit column stride."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{name} must be [rows, K], got {tuple(x.shape)}")
    if x.is_contiguous():
        return x
    if (x.stride(1) != 1 and x.shape[1] > 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap, got strides {x.stride()}")
    return x


def _may_write(out: torch.Tensor, what: str, adds: bool, *inputs: torch.Tensor) -> None:
    """Refuses an `out` whose gradient a call that writes through its address would falsify: one that is overwritten, or a
    leaf or a view of one, where it needs a gradient itself, and any where the inputs do. What is added to an intermediate
    result leaves its gradient as it is."""
    _no_tangents(what, out, *inputs)
    if torch.is_grad_enabled():
        if any(t.requires_grad for t in inputs):
            raise RuntimeError(f"mi355moe: {what} with out= has no gradient, but an input needs one; pass detached inputs, or "
                               "call it under torch.no_grad()")
        if out.requires_grad and (not adds or (out if out._base is None else out._base).is_leaf):
            raise RuntimeError(f"mi355moe: {what} writes out, which needs a gradient; pass out.detach(), or call it under "
                               "torch.no_grad()")


class _NoGradient(torch.autograd.Function):
    """A finished result as an output of inputs that need gradients: the backward pass raises in place of losing them."""

    @staticmethod
    def forward(ctx, out, what, *inputs):
        ctx.what = what
        return out

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError(f"mi355moe: {ctx.what} has no gradient; pass x.detach() and topk_weights.detach() where that is meant")


def _without_gradient(out: torch.Tensor, what: str, *inputs: torch.Tensor) -> torch.Tensor:
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        return _NoGradient.apply(out, what, *inputs)
    return out


def quant_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes uint8 [rows, ceil(K/2)], scales uint8 [rows, ceil(K/32)]) of x [rows, K] (fp32, fp16 or bf16, any row
    stride). A block's scale is the power of two that brings its largest magnitude into [4, 8); values round to nearest
    even and saturate at 6. A block with an infinity or a NaN reads back as NaN."""
    dev = _need_cuda(_rows(x))
    rows, K = x.shape
    dt = weight_dtype_code(x.dtype)
    q = x.new_empty((rows, (K + 1) // 2), dtype=torch.uint8)
    s = x.new_empty((rows, (K + BLOCK - 1) // BLOCK), dtype=torch.uint8)
    with _on_device(dev):
        _lib.check("mi355moe_mxfp4_quant_rows", _lib.lib().mi355moe_mxfp4_quant_rows(
            _addr(x), dt, rows, K, _row_stride(x), _addr(q), _addr(s), _raw_stream(dev)))
    return q, s


def dequant_rows(q: torch.Tensor, scale: torch.Tensor, K: int | None = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, K] of codes [rows, ceil(K/2)] and scales [rows, ceil(K/32)] (K: twice the codes' columns unless
    given). Exact in fp32 and bf16 within their range; fp16 rounds and overflows as a conversion does."""
    dev = _need_cuda(_codes(q, "q"), _codes(scale, "scale"))
    if q.dim() != 2 or scale.dim() != 2:
        raise ValueError("q and scale must be [rows, columns]")
    K = 2 * q.shape[1] if K is None else int(K)
    rows = q.shape[0]
    if K < 1 or q.shape[1] != (K + 1) // 2 or tuple(scale.shape) != (rows, (K + BLOCK - 1) // BLOCK):
        raise ValueError(f"rows of {K} values have {(K + 1) // 2} code and {(K + BLOCK - 1) // BLOCK} scale bytes, got "
                         f"{tuple(q.shape)} and {tuple(scale.shape)}")
    dt = weight_dtype_code(out_dtype)
    q, scale = q.contiguous(), scale.contiguous()
    out = q.new_empty((rows, K), dtype=out_dtype)
    with _on_device(dev):
        _lib.check("mi355moe_mxfp4_dequant_rows", _lib.lib().mi355moe_mxfp4_dequant_rows(
            _addr(q), _addr(scale), rows, K, _addr(out), dt, _raw_stream(dev)))
    return out


@functools.lru_cache(maxsize=4096)
def _matmul_bytes(M: int, N: int, K: int) -> int:
    return _lib.lib().mi355moe_mxfp4_matmul_workspace_bytes(M, N, K)


def _aligned(t: torch.Tensor, nbytes: int) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % nbytes == 0 else t.clone()


def matmul(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """A W^T [M, N] of MXFP4 rows a [M, K/2], a_scale [M, K/32] and w [N, K/2], w_scale [N, K/32]; K % 32 == 0. Products
    are exact and summed in fp32; `out` (fp32, fp16 or bf16, any row stride) is written, not accumulated into."""
    dev = _need_cuda(_codes(a, "a"), _codes(a_scale, "a_scale"), _codes(w, "w"), _codes(w_scale, "w_scale"), out)
    if any(t.dim() != 2 for t in (a, a_scale, w, w_scale)):
        raise ValueError("a, a_scale, w and w_scale must be [rows, columns]")
    M, N, K = a.shape[0], w.shape[0], 2 * a.shape[1]
    if K < BLOCK or K % BLOCK or N < 1:
        raise ValueError(f"K must be a positive multiple of {BLOCK} and N positive, got K {K}, N {N}")
    for name, t, shape in (("a_scale", a_scale, (M, K // BLOCK)), ("w", w, (N, K // 2)), ("w_scale", w_scale, (N, K // BLOCK))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: expected {shape}, got {tuple(t.shape)}")
    given = out is not None
    if given:
        _may_write(out, "mxfp4.matmul", False)
    else:
        out = a.new_empty((M, N), dtype=out_dtype)
    dt = weight_dtype_code(out.dtype)
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out must be {(M, N)}, got {tuple(out.shape)}")
    _rows(out, "out")
    if M == 0:
        return out
    a, w = _aligned(a, 16), _aligned(w, 16)
    a_scale, w_scale = _aligned(a_scale, 4), _aligned(w_scale, 4)
    L = _lib.lib()
    nb = _matmul_bytes(M, N, K)
    if nb < 0:
        raise ValueError(f"mi355moe_mxfp4_matmul: unsupported size M {M}, N {N}, K {K}")
    with _on_device(dev):
        ws = a.new_empty(nb) if nb else None
        _lib.check("mi355moe_mxfp4_matmul", L.mi355moe_mxfp4_matmul(
            _addr(a), _addr(a_scale), M, _addr(w), _addr(w_scale), N, K, _addr(out), dt, _row_stride(out), _addr(ws), nb, _raw_stream(dev)))
    if given:
        increment_version(out)
    return out


def _arranged(scale: torch.Tensor) -> torch.Tensor:
    """Scales [n, rows, K/32] in the order the expert products read them (steps of 256 columns of neighbouring rows)."""
    n, rows, K = scale.shape[0], scale.shape[1], scale.shape[2] * BLOCK
    dev = _need_cuda(scale)
    L = _lib.lib()
    out = torch.empty(n, -(-K // 256), rows, 8, dtype=torch.uint8, device=dev)
    with _on_device(dev):
        _lib.check("mi355moe_mxfp4_arrange_scales",
                   L.mi355moe_mxfp4_arrange_scales(_addr(scale), n, rows, K, _addr(out), _raw_stream(dev)))
    return out


class Mxfp4Experts:
    """A layer's MXFP4 experts plus the C descriptor. The codes stay the caller's tensors; the scales are copied once (later
    changes of the caller's do not reach them) into the order the kernels read, a seventeenth of the layer's bytes.
    arrange=False keeps the caller's, which needs H and I to be multiples of 128 and costs 0 to 6 % of a call (hidden 4096,
    intermediate 1024, 288 experts, top-8: 8 tokens 78 us arranged and 83 as they come, 64 tokens 286 and 296, 2047 tokens
    547 and 555). Built on the current stream: as with any tensor, another stream waits for it before its first call."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
                 arrange: bool = True):
        for name, t in (("w13", w13), ("w13_scale", w13_scale), ("w2", w2), ("w2_scale", w2_scale)):
            _codes(t, name)
            if t.dim() != 3:
                raise ValueError(f"{name} must be [n, rows, columns], got {tuple(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if t.device != w13.device:
                raise ValueError(f"{name} is on {t.device}, w13 on {w13.device}")
        n, I2, H = w13.shape[0], w13.shape[1], 2 * w13.shape[2]
        I = I2 // 2
        if n < 1 or I2 % 2 or H < BLOCK or H % BLOCK or I < BLOCK or I % BLOCK:
            raise ValueError(f"w13 must be [n, 2I, H/2] with H and I multiples of {BLOCK}, got {tuple(w13.shape)}")
        for name, t, shape in (("w2", w2, (n, H, I // 2)), ("w13_scale", w13_scale, (n, 2 * I, H // BLOCK)),
                               ("w2_scale", w2_scale, (n, H, I // BLOCK))):
            if tuple(t.shape) != shape:
                raise ValueError(f"{name}: expected {shape}, got {tuple(t.shape)}")
        for name, t, by in (("w13", w13, 16), ("w2", w2, 16), ("w13_scale", w13_scale, 1 if arrange else 4),
                            ("w2_scale", w2_scale, 1 if arrange else 4)):
            if t.data_ptr() % by:
                raise ValueError(f"{name} must lie at a {by}-byte address")
        if not arrange and (H % 128 or I % 128):
            raise ValueError(f"scales are used as they are only for H and I that are multiples of 128, got {H} and {I}")
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.n, self.K, self.N = n, H, I
        self._bytes: dict = {}
        self._s13, self._s2 = (_arranged(w13_scale), _arranged(w2_scale)) if arrange else (w13_scale, w2_scale)
        d = _lib.Mxfp4LayerDesc()
        d.n, d.hidden, d.intermediate, d.arranged = n, H, I, int(arrange)
        d.w13, d.w13_scale = ctypes.c_void_p(w13.data_ptr()), ctypes.c_void_p(self._s13.data_ptr())
        d.w2, d.w2_scale = ctypes.c_void_p(w2.data_ptr()), ctypes.c_void_p(self._s2.data_ptr())
        self.desc = d

    @classmethod
    def from_dense(cls, w13: torch.Tensor, w2: torch.Tensor) -> "Mxfp4Experts":
        """Quantise dense experts w13 [n, 2I, H] and w2 [n, H, I] (fp32, fp16 or bf16)."""
        if w13.dim() != 3 or w2.dim() != 3:
            raise ValueError("w13 and w2 must be [n, rows, columns]")
        out = []
        for w in (w13, w2):
            q, s = quant_rows(w.reshape(-1, w.shape[-1]))
            out += [q.reshape(*w.shape[:2], -1), s.reshape(*w.shape[:2], -1)]
        return cls(*out)

    @property
    def device(self) -> torch.device:
        return self.w13.device

    def workspace_bytes(self, T: int, topk: int) -> int:
        """The scratch a call of T tokens takes (-1: more than a call can have)."""
        nb = self._bytes.get((T, topk))
        if nb is None:
            nb = self._bytes[T, topk] = _lib.lib().mi355moe_mxfp4_moe_workspace_bytes(ctypes.byref(self.desc), T, topk)
        return nb

    def expert_bytes(self) -> int:
        """Bytes of one expert's three matrices and their block scales."""
        return 3 * self.K * self.N * 17 // 32


def _pairs(t: torch.Tensor, T: int) -> torch.Tensor:
    return t if t.dim() == 2 and t.is_contiguous() else t.reshape(T, -1).contiguous()


def moe_forward_ids(experts: Mxfp4Experts, x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                    limit: float = 10.0, expert_map: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None, accumulate: bool = False) -> torch.Tensor:
    """Routed-expert output [T, H] in x's dtype (unless out / out_dtype say otherwise). x: fp32, fp16 or bf16 [T, H];
    topk_ids int32/int64 [T, k] (global ids; expert_map maps them to local ids or -1; pairs of no local expert are
    skipped); topk_weights [T, k] (already scaled by the router). accumulate: out, which then has to be given, += the
    routed sum with one rounding (out holds the shared expert's output, and may be an intermediate result of autograd's: its
    own gradient passes through). The routed experts have no gradient: where x or topk_weights need one, out is refused and
    the result's backward raises; pass detached ones."""
    dev = _need_cuda(x, topk_ids, topk_weights, expert_map, out)
    if dev != experts.device:
        raise ValueError(f"activations on {dev}, experts on {experts.device}")
    if x.dim() != 2 or x.shape[1] != experts.K:
        raise ValueError(f"x must be [T, {experts.K}], got {tuple(x.shape)}")
    if expert_map is not None and expert_map.numel() == 0:
        raise ValueError("expert_map has no entries")        # (its address would read as no map: ids taken as local ones)
    _rows(x)
    T = x.shape[0]
    if topk_ids.dim() not in (1, 2) or topk_ids.shape[0] != T or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_ids and topk_weights must be [T, k]")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    given = out is not None
    if given:
        _may_write(out, "mxfp4.moe_forward_ids", accumulate, x, topk_weights)
    else:
        _no_tangents("mxfp4.moe_forward_ids", x, topk_weights)
        out = x.new_empty((T, experts.K), dtype=out_dtype or x.dtype)
    if tuple(out.shape) != (T, experts.K):
        raise ValueError(f"out must be [T, {experts.K}], got {tuple(out.shape)}")
    _rows(out, "out")
    xdt, odt = weight_dtype_code(x.dtype), weight_dtype_code(out.dtype)
    if T == 0:
        return out
    ids, w = _pairs(topk_ids, T), _pairs(topk_weights, T)
    topk = ids.shape[1]
    L = _lib.lib()
    nb = experts.workspace_bytes(T, topk)
    if nb < 0:
        raise ValueError(f"mi355moe_mxfp4_moe_forward_ids: unsupported size (T {T}, top-{topk})")
    em = None if expert_map is None else expert_map.to(torch.int64).contiguous()
    with _on_device(dev):
        ws = experts.w13.new_empty(nb)
        _lib.check("mi355moe_mxfp4_moe_forward_ids", L.mi355moe_mxfp4_moe_forward_ids(
            ctypes.byref(experts.desc), _addr(x), xdt, _row_stride(x), T, _addr(ids), ids_dtype_code(ids.dtype), _addr(w),
            weight_dtype_code(w.dtype), topk, _addr(em), 0 if em is None else em.numel(), float(limit), _addr(out), odt,
            _row_stride(out), _lib.OPT_ACCUMULATE if accumulate else 0, _addr(ws), ws.numel(), _raw_stream(dev)))
    if given:
        increment_version(out)
        return out
    return _without_gradient(out, "mxfp4.moe_forward_ids", x, topk_weights)


def fused_experts_mxfp4(hidden: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
                        topk_ids: torch.Tensor, scales: tuple, *, limit: float = 10.0,
                        expert_map: torch.Tensor | None = None) -> torch.Tensor:
    """apply(hidden, w13, w2, topk_weights, topk_ids, scales) for MXFP4 experts: scales = (w13_scale, w2_scale). Hosts
    that call it often keep an Mxfp4Experts and call moe_forward_ids: this form reads the scales as they are, and arranges
    them in every call where hidden or intermediate is no multiple of 128."""
    whole = (2 * w13.shape[-1]) % 128 == 0 and (2 * w2.shape[-1]) % 128 == 0
    return moe_forward_ids(Mxfp4Experts(w13, scales[0], w2, scales[1], arrange=not whole), hidden, topk_ids, topk_weights,
                           limit=limit, expert_map=expert_map, out_dtype=hidden.dtype)
