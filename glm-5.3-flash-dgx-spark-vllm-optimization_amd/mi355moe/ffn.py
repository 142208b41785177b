"""The gated feed-forward block of a layer's shared expert and the dense product with its epilogue, with their gradients.

    [g | u] = x W13^T;  h = silu(min(g, L)) * clamp(u, -L, L)   (the limit iff L != 0)

in fp16 or bf16 with fp32 sums and one rounding: both projections, the activation and the product. The
shared expert is h W2^T (`linear`, which can add the residual stream to it); its output is what the routed experts'
`accumulate` adds to.

    out = act(x W^T + bias) + residual

in the same types, likewise rounded once: a dense product with its epilogue.

  gated            h, differentiable in x and w13
  gated_forward    h, or h and the fp32 [g | u] that the gradient reads
  gated_backward   (dx, dw13) from dh and [g | u]
  linear           out, differentiable in x, w, bias and residual
  linear_forward   out, or out and the fp32 z = x W^T + bias that the gradient reads
  linear_backward  (dx, dw, dbias) from dout and z

The gradient reads g and u in fp32 (8 bytes per token and column, kept from the forward pass): read back they cost a
fifth of the time that computing them again would, and the gradients carry one rounding less than with 16-bit copies.
Every call runs on the current stream of its tensors' device; scratch comes from torch's caching allocator.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import (_addr, _capturing, _current_device, _need_cuda, _no_tangents, _on_device, _once, _packed, _plain,
                  _raw_stream, _row_stride, _rows_any, _stream_at, act_dtype_code, weight_dtype_code)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t [rows, K] itself where its rows lie apart at 16-byte addresses, at most 2^22 values from one to the next, else a
    contiguous copy."""
    if t.is_contiguous() and t.shape[1] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    if t.stride(1) == 1 and (t.shape[0] <= 1 or (t.shape[1] <= t.stride(0) <= 1 << 22 and t.stride(0) % 8 == 0)) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=4096)
def _forward_bytes(T: int, H: int, I: int) -> int:
    return _lib.lib().mi355moe_gated_forward_workspace_bytes(T, H, I)


@functools.lru_cache(maxsize=4096)
def _backward_bytes(T: int, H: int, I: int) -> int:
    return _lib.lib().mi355moe_gated_backward_workspace_bytes(T, H, I)


def _check(x: torch.Tensor, w13: torch.Tensor) -> tuple[torch.device, int]:
    dev = _need_cuda(x, w13)
    _no_tangents("the gated block", x, w13)
    code = act_dtype_code(x.dtype)
    if w13.dtype != x.dtype:
        raise ValueError(f"x is {x.dtype}, w13 {w13.dtype}")
    if w13.dim() != 2 or w13.shape[0] % 16 or w13.shape[1] % 8 or w13.numel() == 0:
        raise ValueError(f"w13 must be [2I, H] with I and H multiples of 8, got {tuple(w13.shape)}")
    if x.dim() < 1 or x.shape[-1] != w13.shape[1]:
        raise ValueError(f"x must be [..., {w13.shape[1]}], got {tuple(x.shape)}")
    return dev, code


def gated_forward(x: torch.Tensor, w13: torch.Tensor, limit: float = 0.0, save: bool = False):
    """h [..., I] of x [..., H] and w13 [2I, H] (gate rows, then up rows), or with save (h, gu), gu fp32 [rows, 2I] = x
    W13^T for gated_backward. No gradient is recorded."""
    dev, code = _check(x, w13)
    I, H = w13.shape[0] // 2, w13.shape[1]
    x, w13 = _plain(x), _plain(w13)
    x2 = _rows16(x if x.dim() == 2 else x.reshape(-1, H))
    w = _rows16(w13) if w13.is_contiguous() else w13.contiguous()
    T = x2.shape[0]
    with _on_device(dev):
        h = x2.new_empty((T, I))
        gu = x2.new_empty((T, 2 * I), dtype=torch.float32) if save else None
        nb = _forward_bytes(T, H, I)
        ws = x2.new_empty(nb, dtype=torch.uint8) if nb > 0 else None
        _lib.check("mi355moe_gated_forward", _lib.lib().mi355moe_gated_forward(
            _addr(x2), code, T, H, _row_stride(x2), _addr(w), I, float(limit), _addr(h), I, _addr(gu), _addr(ws), max(nb, 0),
            _raw_stream(dev)))
    if x.dim() != 2:
        h = h.reshape(*x.shape[:-1], I)
    return (h, gu) if save else h


def gated_backward(dh: torch.Tensor, gu: torch.Tensor, x: torch.Tensor, w13: torch.Tensor, limit: float = 0.0,
                   need_dx: bool = True, need_dw13: bool = True):
    """(dx, dw13) in x's dtype (None where not needed) from dh [..., I], the forward's gu fp32 [rows, 2I], x and w13.
    Each gradient is a fp32 sum over [dg | du] rounded to x's dtype; the sums' order does not vary."""
    dev, code = _check(x, w13)
    _need_cuda(x, dh, gu)
    _no_tangents("the gated block's backward", dh, gu)
    I, H = w13.shape[0] // 2, w13.shape[1]
    if dh.dtype != x.dtype or dh.shape[:-1] != x.shape[:-1] or dh.shape[-1] != I:
        raise ValueError(f"dh must be {x.dtype} {(*x.shape[:-1], I)}, got {dh.dtype} {tuple(dh.shape)}")
    x2, d2, w = _plain(x), _plain(dh), _plain(w13)
    if x.dim() != 2:
        x2, d2 = x2.reshape(-1, H), d2.reshape(-1, I)
    T = x2.shape[0]
    if gu.dtype != torch.float32 or tuple(gu.shape) != (T, 2 * I) or not gu.is_contiguous():
        raise ValueError(f"gu must be contiguous float32 {(T, 2 * I)}, got {gu.dtype} {tuple(gu.shape)}")
    x2, d2 = _rows16(x2), _rows16(d2)
    w = _rows16(w) if w.is_contiguous() else w.contiguous()
    with _on_device(dev):
        dx = x2.new_empty((T, H)) if need_dx else None
        if T == 0:
            return (dx.reshape(x.shape) if need_dx else None, w.new_zeros(w13.shape) if need_dw13 else None)
        dw = x2.new_empty((2 * I, H)) if need_dw13 else None
        nb = _backward_bytes(T, H, I)
        ws = x2.new_empty(max(nb, 0), dtype=torch.uint8)
        _lib.check("mi355moe_gated_backward", _lib.lib().mi355moe_gated_backward(
            _addr(d2), _row_stride(d2), _addr(gu), _addr(x2), code, T, H, _row_stride(x2), _addr(w), I, float(limit), _addr(dx), _addr(dw),
            _addr(ws), max(nb, 0), _raw_stream(dev)))
    return (dx if dx is None or x.dim() == 2 else dx.reshape(x.shape)), dw


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, limit):
        h, gu = gated_forward(x, w13, limit, save=True)
        ctx.save_for_backward(x, w13, gu)
        ctx.limit = limit
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        if _capturing(dh.device):
            raise RuntimeError("mi355moe: the backward pass of an eagerly recorded ffn.gated cannot be captured; capture "
                               "ffn.gated_forward(save=True) and ffn.gated_backward")
        x, w13, gu = ctx.saved_tensors
        dx, dw = gated_backward(dh, gu, x, w13, ctx.limit, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None


def gated(x: torch.Tensor, w13: torch.Tensor, limit: float = 0.0) -> torch.Tensor:
    """h [..., I] = silu(min(g, L)) * clamp(u, -L, L) of x [..., H] and w13 [2I, H], differentiable once in x and w13
    by reverse mode (forward-mode derivatives are refused). While a graph is captured, a call that would record a gradient is
    refused: torch's autograd does not keep an eager graph of the same leaves apart from a captured one; capture
    gated_forward(save=True) and gated_backward instead. The backward pass of an eager call is refused during capture too."""
    if torch.is_grad_enabled() and (x.requires_grad or w13.requires_grad):
        dev, _ = _check(x, w13)
        if _capturing(dev):
            raise RuntimeError("mi355moe: gated cannot record a gradient during graph capture; capture "
                               "ffn.gated_forward(save=True) and ffn.gated_backward")
        return _Gated.apply(x, w13, float(limit))
    return gated_forward(x, w13, limit)


ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


@functools.lru_cache(maxsize=4096)
def _linear_bytes(M: int, K: int, N: int) -> int:
    return _lib.lib().mi355moe_linear_forward_workspace_bytes(M, K, N)


@functools.lru_cache(maxsize=4096)
def _linear_grad_bytes(*call) -> int:
    return _lib.lib().mi355moe_linear_backward_call_bytes(*call)


def _linear_operand(t: torch.Tensor, K: int) -> tuple[torch.Tensor, int]:
    """t [..., K] as the product reads its rows, and the values from one row to the next: where K is a multiple of 8 the rows lie
    at 16-byte addresses."""
    if K & 7:
        return _rows_any(t)
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t, K
    t = _plain(t)
    t = _rows16(t if t.dim() == 2 else t.reshape(-1, K))
    return t, _row_stride(t)


def _check_linear(x, w, bias, activation, residual):
    dev = _need_cuda(x, w, bias, residual)
    _no_tangents("the dense product", x, w, bias, residual)
    code = act_dtype_code(x.dtype)
    if w.dtype != x.dtype:
        raise ValueError(f"x is {x.dtype}, w {w.dtype}")
    shape, ws = x.shape, w.shape
    if len(ws) != 2 or w.numel() == 0:
        raise ValueError(f"w must be [N, K], got {tuple(ws)}")
    if not shape or shape[-1] != ws[1]:
        raise ValueError(f"x must be [..., {ws[1]}], got {tuple(shape)}")
    if bias is not None and bias.shape != ws[:1]:
        raise ValueError(f"bias must be {(ws[0],)}, got {tuple(bias.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != (*shape[:-1], ws[0])):
        raise ValueError(f"residual must be {x.dtype} {(*shape[:-1], ws[0])}, got {residual.dtype} {tuple(residual.shape)}")
    return dev, code, _lib.F32 if bias is None else weight_dtype_code(bias.dtype)


def linear_forward(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                   residual: torch.Tensor | None = None, save: bool = False):
    """out [..., N] of x [..., K] and w [N, K], or with save (out, z), z fp32 [rows, N] = x W^T + bias for linear_backward (None
    without an activation, whose gradient does not read it). No gradient is recorded."""
    return _linear(_check_linear(x, w, bias, activation, residual), x, w, bias, activation, residual, save)


def _linear(kinds, x, w, bias, activation, residual, save):
    """linear_forward of arguments that have been looked at (kinds: what _check_linear said of them)."""
    dev, code, bcode = kinds
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _linear(kinds, x, w, bias, activation, residual, save)
    N, K = w.shape
    (x2, ldx), (w2, ldw) = _linear_operand(x, K), _linear_operand(w, K)
    b = None if bias is None else _packed(bias)
    r, ldr = (residual, N) if residual is None or residual.is_contiguous() else _rows_any(residual)
    M = x2.numel() // K
    out = x2.new_empty(M, N) if x.dim() == 2 else x2.new_empty((*x.shape[:-1], N))
    z = x2.new_empty(M, N, dtype=torch.float32) if save and activation is not None else None
    nb = _linear_bytes(M, K, N)
    ws = x2.new_empty(nb, dtype=torch.uint8) if nb > 0 else None
    rc = _lib.lib().mi355moe_linear_forward(
        x2.data_ptr(), code, M, K, ldx, w2.data_ptr(), N, ldw, _addr(b), bcode, ACTIVATIONS[activation], _addr(r), ldr, out.data_ptr(), N,
        _addr(z), _addr(ws), max(nb, 0), _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_linear_forward", rc)
    return (out, z) if save else out


def linear_backward(dout: torch.Tensor, z: torch.Tensor | None, x: torch.Tensor, w: torch.Tensor, activation: str | None = None,
                    bias_dtype: torch.dtype | None = None, need_dx: bool = True, need_dw: bool = True):
    """(dx, dw, dbias) from dout [..., N], the forward's z, x and w: fp32 sums, dx and dw in x's dtype, dbias in bias_dtype (None
    where there is no bias or the gradient is not needed); the sums' order does not vary. With a curved activation dz = dout act'(z)
    is rounded once to x's dtype for the two products (dbias sums it unrounded). x's values are read for dw, w's for dx. residual's
    gradient is dout."""
    kinds = _check_linear(x, w, None, activation, None)
    _need_cuda(x, dout, z)
    _no_tangents("the dense product's backward", dout, z)
    N = w.shape[0]
    if dout.dtype != x.dtype or dout.shape != (*x.shape[:-1], N):
        raise ValueError(f"dout must be {x.dtype} {(*x.shape[:-1], N)}, got {dout.dtype} {tuple(dout.shape)}")
    if bias_dtype is not None:
        weight_dtype_code(bias_dtype)
    M = dout.numel() // N
    if activation is not None and (z is None or z.dtype != torch.float32 or tuple(z.shape) != (M, N) or not z.is_contiguous()):
        raise ValueError(f"z must be contiguous float32 {(M, N)}, got {None if z is None else (z.dtype, tuple(z.shape))}")
    return _linear_grads(kinds, dout, z, x, w, activation, bias_dtype, need_dx, need_dw)


def _linear_grads(kinds, dout, z, x, w, activation, bias_dtype, need_dx, need_dw):
    """linear_backward of arguments that have been looked at; x may be None without dw, w without dx, z without any of the three. (It
    runs on autograd's own thread, where a helper's frame costs some us.)"""
    dev, code, _ = kinds
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _linear_grads(kinds, dout, z, x, w, activation, bias_dtype, need_dx, need_dw)
    N = dout.shape[-1]
    K = w.shape[1] if w is not None else 1 if x is None else x.shape[-1]         # (the bias' gradient alone: any K)
    M = dout.numel() // N
    dx = dw = None
    if need_dx:
        dx = torch.empty_like(x) if x is not None and x.is_contiguous() else dout.new_empty((*dout.shape[:-1], K))
    if need_dw:
        dw = torch.empty_like(w) if w is not None and w.is_contiguous() else dout.new_empty(N, K)
    db = None if bias_dtype is None else dout.new_empty(N, dtype=bias_dtype)
    if M == 0 or (dx is None and dw is None and db is None):
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    # (x is read for dw, w for dx: what is not read is not copied to where it could be)
    x2, ldx = _linear_operand(x, K) if need_dw else (None, (K + 7) & ~7)
    w2, ldw = _linear_operand(w, K) if need_dx else (None, (K + 7) & ~7)
    d2, ldd = (dout, N) if dout.is_contiguous() else _rows_any(dout)
    at = d2.data_ptr()
    nb = _linear_grad_bytes(M, K, N, code, ACTIVATIONS[activation], not at & 15 and not ldd & 7 and ldd <= 1 << 22, need_dx, need_dw, db is not None)
    ws = dout.new_empty(nb, dtype=torch.uint8) if nb > 0 else None
    rc = _lib.lib().mi355moe_linear_backward(
        at, ldd, None if activation is None else z.data_ptr(), x2 if x2 is None else x2.data_ptr(), code, M, K, ldx,
        w2 if w2 is None else w2.data_ptr(), N, ldw, ACTIVATIONS[activation], dx if dx is None else dx.data_ptr(), dw if dw is None else dw.data_ptr(),
        db if db is None else db.data_ptr(), _lib.F32 if db is None else weight_dtype_code(bias_dtype), ws if ws is None else ws.data_ptr(), max(nb, 0),
        _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_linear_backward", rc)
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, kinds, activation):
        # what the gradients that are asked for read: x for w's, w for x's, z for these and the bias', nothing for the residual's
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need_z = need_x or need_w or need_b
        out = _linear(kinds, x, w, bias, activation, residual, need_z)
        out, z = out if need_z else (out, None)
        ctx.save_for_backward(x if need_w else None, w if need_x else None, z)
        ctx.rest = kinds, activation, None if bias is None else bias.dtype
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        if _capturing(ctx.rest[0][0]):
            raise RuntimeError("mi355moe: the backward pass of an eagerly recorded ffn.linear cannot be captured; capture "
                               "ffn.linear_forward(save=True) and ffn.linear_backward")
        x, w, z = ctx.saved_tensors
        kinds, activation, bias_dtype = ctx.rest
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            dx, dw, db = _linear_grads(kinds, dout, z, x, w, activation, bias_dtype if need[2] else None, need[0], need[1])
        return dx, dw, db, dout if need[3] else None, None, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """out [..., N] = act(x W^T + bias) + residual of x [..., K], w [N, K], bias [N] (any of fp32, fp16, bf16) and residual [..., N];
    activation None, "relu", "silu", "gelu" or "gelu_tanh". Where K is a multiple of 8, an x or w whose rows lie at other than 16-byte
    addresses is copied in every call: keep weights packed. Differentiable once in the four tensors by reverse mode
    (forward-mode derivatives are refused). While a graph is captured, a call that would record a gradient, and the backward
    pass of an eager one, are refused; capture linear_forward(save=True) and linear_backward instead."""
    kinds = _check_linear(x, w, bias, activation, residual)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        if _capturing(kinds[0]):
            raise RuntimeError("mi355moe: linear cannot record a gradient during graph capture; capture "
                               "ffn.linear_forward(save=True) and ffn.linear_backward")
        return _Linear.apply(x, w, bias, residual, kinds, activation)
    return _linear(kinds, x, w, bias, activation, residual, False)
