"""The gated feed-forward block of a layer's shared expert and its gradient.

    [g | u] = x W13^T;  h = silu(min(g, L)) * clamp(u, -L, L)   (the limit iff L != 0)

in fp16 or bf16 with fp32 sums and one rounding: both projections, the activation and the product. The
shared expert is h W2^T (a plain library product); its output is what the routed experts' `accumulate` adds to.

  gated            h, differentiable in x and w13
  gated_forward    h, or h and the fp32 [g | u] that the gradient reads
  gated_backward   (dx, dw13) from dh and [g | u]

The gradient reads g and u in fp32 (8 bytes per token and column, kept from the forward pass): read back they cost a
fifth of the time that computing them again would, and the gradients carry one rounding less than with 16-bit copies.
Every call runs on the current stream of its tensors' device; scratch comes from torch's caching allocator.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _addr, _capturing, _need_cuda, _no_tangents, _on_device, _raw_stream, act_dtype_code


def _row_stride(t: torch.Tensor) -> int:
    """Values between two rows of t. One row (or none) has none: its stride(0) can be anything, also in what torch calls
    contiguous."""
    return t.shape[1] if t.shape[0] <= 1 else t.stride(0)


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


def _plain(t: torch.Tensor) -> torch.Tensor:
    return t.detach() if t.requires_grad else t


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
