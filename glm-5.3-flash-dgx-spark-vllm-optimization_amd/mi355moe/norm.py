"""The norms before and after a block, with its gate and the scaled residual sum, with gradients.

    u = branch * r(branch) * post          (branch itself without post)
    s = residual_scale * residual + scale * gate * u
    y = s * r(s) * pre                     r(v) = 1 / sqrt(mean of v^2 over the last dimension + eps)

  join           (s, y), or s alone without pre: what stands between two blocks, in one pass over the rows
  rms            y of one tensor: the norm before the first block
  join_forward, join_backward   the explicit pair (for capture)

Everything is fp32 from the loads to one rounding of s and of y; y goes by s before its rounding. The gradients form s again
from the inputs in fp32, and keep two fp32 numbers a row from the forward pass. Rows are fp32, fp16 or bf16. Values whose squares'
mean leaves fp32's range (magnitudes above 1e19; with eps 0 also rows all below 1e-19) are outside the operator's range. Every call
runs on the current stream of its tensors' device; outputs and scratch come from torch's caching allocator.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .ops import (_capturing, _current_device, _empty_like, _need_cuda, _no_tangents, _once, _packed, _rows_any, _stream_at,
                  weight_dtype_code)

_NONE, _CHANNEL, _TOKEN, _FULL = 0, 1, 2, 3


@functools.lru_cache(maxsize=4096)
def _backward_bytes(rows: int, H: int) -> int:
    return _lib.lib().mi355moe_norm_backward_workspace_bytes(rows, H)


def _gate_kind(shape: torch.Size, gate: torch.Size) -> int:
    if gate == shape:
        return _FULL
    if gate == shape[-1:]:
        return _CHANNEL
    if gate == (*shape[:-1], 1):
        return _TOKEN
    raise ValueError(f"gate must be {(shape[-1],)}, {(*shape[:-1], 1)} or {tuple(shape)}, got {tuple(gate)}")


def _check(branch, residual, post, gate, pre):
    dev = _need_cuda(branch, residual, post, gate, pre)
    _no_tangents("the norms around a block", branch, residual, post, gate, pre)
    dtype, shape = branch.dtype, branch.shape
    code = weight_dtype_code(dtype)
    if not shape or shape[-1] == 0:
        raise ValueError(f"branch must be [..., H], got {tuple(shape)}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype):
        raise ValueError(f"residual must be {dtype} {tuple(shape)}, got {residual.dtype} {tuple(residual.shape)}")
    wcode = _lib.F32
    for w in (post, pre):
        if w is not None:
            wcode = weight_dtype_code(w.dtype)
            if w.shape != shape[-1:]:
                raise ValueError(f"{'post' if w is post else 'pre'} must be {(shape[-1],)}, got {tuple(w.shape)}")
    if post is not None and pre is not None and post.dtype != pre.dtype:
        raise ValueError(f"post is {post.dtype}, pre {pre.dtype}")
    if gate is None:
        return dev, code, wcode, _NONE, _lib.F32
    return dev, code, wcode, _gate_kind(shape, gate.shape), weight_dtype_code(gate.dtype)


# The two functions below run once a step, the second on autograd's own thread, where what the first thread touched last is far
# away: a helper's frame there costs some us. So what is there already is looked at in place, and helpers take the rest.


def _forward(kinds, branch, residual, post, gate, pre, eps, scale, residual_scale, need_s, need_stats):
    dev, code, wcode, kind, gcode = kinds
    if pre is None and not need_s:
        raise ValueError("neither s nor y is asked for")
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _forward(kinds, branch, residual, post, gate, pre, eps, scale, residual_scale, need_s, need_stats)
    H = branch.shape[-1]
    n = branch.numel() // H
    s = _empty_like(branch) if need_s else None
    y = _empty_like(branch) if pre is not None else None
    stats = branch.new_empty(n, 2, dtype=torch.float32) if need_stats else None
    if n:
        b, ldb = (branch, H) if branch.is_contiguous() else _rows_any(branch)
        r, ldr = (residual, H) if residual is None or residual.is_contiguous() else _rows_any(residual)
        post = post if post is None or post.is_contiguous() else _packed(post)
        pre = pre if pre is None or pre.is_contiguous() else _packed(pre)
        gate = gate if gate is None or gate.is_contiguous() else _packed(gate)
        rc = _lib.lib().mi355moe_norm_forward(
            b.data_ptr(), code, n, H, ldb, r if r is None else r.data_ptr(), ldr, post if post is None else post.data_ptr(),
            pre if pre is None else pre.data_ptr(), wcode, gate if gate is None else gate.data_ptr(), gcode, kind, eps, scale,
            residual_scale, s if s is None else s.data_ptr(), y if y is None else y.data_ptr(),
            stats if stats is None else stats.data_ptr(), _stream_at(dev.index))
        if rc:
            _lib.check("mi355moe_norm_forward", rc)
    return s, y, stats


def join_forward(branch: torch.Tensor, residual: torch.Tensor | None = None, post: torch.Tensor | None = None,
                 gate: torch.Tensor | None = None, pre: torch.Tensor | None = None, eps: float = 1e-6, scale: float = 1.0,
                 residual_scale: float = 1.0, need_s: bool = True):
    """(s, y, stats): s and y as join has them (None where there is none), stats fp32 [rows, 2] for join_backward. No gradient is
    recorded."""
    return _forward(_check(branch, residual, post, gate, pre), branch, residual, post, gate, pre, float(eps), float(scale),
                    float(residual_scale), need_s, True)


def join_backward(ds: torch.Tensor | None, dy: torch.Tensor | None, stats: torch.Tensor, branch: torch.Tensor,
                  residual: torch.Tensor | None = None, post: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  pre: torch.Tensor | None = None, scale: float = 1.0, residual_scale: float = 1.0,
                  need: tuple = (True, True, True, True, True)):
    """(dbranch, dresidual, dpost, dgate, dpre) from ds and dy (None: zero), the forward's stats and its inputs, each shaped and
    typed like its input; None where the input is, or `need` (in that order) says no."""
    kinds = _check(branch, residual, post, gate, pre)
    _need_cuda(branch, ds, dy, stats)
    _no_tangents("the norms' backward", ds, dy)
    for name, d in (("ds", ds), ("dy", dy)):
        if d is not None and (d.dtype != branch.dtype or d.shape != branch.shape):
            raise ValueError(f"{name} must be {branch.dtype} {tuple(branch.shape)}, got {d.dtype} {tuple(d.shape)}")
    if dy is not None and pre is None:
        raise ValueError("dy without pre")
    n = branch.numel() // branch.shape[-1]
    if stats.dtype != torch.float32 or tuple(stats.shape) != (n, 2) or not stats.is_contiguous():
        raise ValueError(f"stats must be contiguous float32 {(n, 2)}, got {stats.dtype} {tuple(stats.shape)}")
    need = (need[0], need[1] and residual is not None, *need[2:])
    return _backward(kinds, ds, dy, stats, branch, residual, post, gate, pre, float(scale), float(residual_scale), need)


def _backward(kinds, ds, dy, stats, branch, residual, post, gate, pre, scale, residual_scale, need):
    """join_backward of arguments that have been looked at (kinds: what _check said of them). residual's values are read with dy only;
    without dy, need[1] alone says whether there is one."""
    dev, code, wcode, kind, gcode = kinds
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _backward(kinds, ds, dy, stats, branch, residual, post, gate, pre, scale, residual_scale, need)
    H = branch.shape[-1]
    n = branch.numel() // H
    db = dr = dpost = dgate = dpre = None
    if need[0]:
        db = torch.empty_like(branch) if branch.is_contiguous() else _empty_like(branch)
    if need[1]:
        dr = torch.empty_like(branch) if branch.is_contiguous() else _empty_like(branch)      # (of branch's shape and type)
    if need[2] and post is not None:
        dpost = torch.empty_like(post) if post.is_contiguous() else _empty_like(post)
    if need[3] and gate is not None:
        dgate = torch.empty_like(gate) if gate.is_contiguous() else _empty_like(gate)
    if need[4] and pre is not None:
        dpre = torch.empty_like(pre) if pre.is_contiguous() else _empty_like(pre)
    if n == 0 or (ds is None and dy is None):
        return tuple(None if t is None else t.zero_() for t in (db, dr, dpost, dgate, dpre))
    if dy is None and dpre is not None:
        dpre.zero_()
    b, ldb = (branch, H) if branch.is_contiguous() else _rows_any(branch)
    if dy is None:
        residual = None
    r, ldr = (residual, H) if residual is None or residual.is_contiguous() else _rows_any(residual)
    s, lds = (ds, H) if ds is None or ds.is_contiguous() else _rows_any(ds)
    y, ldy = (dy, H) if dy is None or dy.is_contiguous() else _rows_any(dy)
    post = post if post is None or post.is_contiguous() else _packed(post)
    pre = pre if pre is None or pre.is_contiguous() else _packed(pre)
    gate = gate if gate is None or gate.is_contiguous() else _packed(gate)
    wpre = None if dy is None else dpre
    nb, ws = 0, None
    if dpost is not None or wpre is not None or (dgate is not None and kind == _CHANNEL):
        nb = _backward_bytes(n, H)
        ws = b.new_empty(max(nb, 0), dtype=torch.uint8)
    rc = _lib.lib().mi355moe_norm_backward(
        s if s is None else s.data_ptr(), lds, y if y is None else y.data_ptr(), ldy, b.data_ptr(), code, n, H, ldb,
        r if r is None else r.data_ptr(), ldr, post if post is None else post.data_ptr(), pre if pre is None else pre.data_ptr(), wcode,
        gate if gate is None else gate.data_ptr(), gcode, kind, scale, residual_scale, stats.data_ptr(),
        db if db is None else db.data_ptr(), dr if dr is None else dr.data_ptr(), dpost if dpost is None else dpost.data_ptr(),
        wpre if wpre is None else wpre.data_ptr(), dgate if dgate is None else dgate.data_ptr(),
        ws if ws is None else ws.data_ptr(), nb if nb > 0 else 0, _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_norm_backward", rc)
    return db, dr, dpost, dgate, dpre


class _Join(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, post, gate, pre, kinds, eps, scale, residual_scale, need_s):
        s, y, stats = _forward(kinds, branch, residual, post, gate, pre, eps, scale, residual_scale, need_s, True)
        # (the residual is read for the gradient of the norm behind the sum; the residual stream of a sum alone may go on in place)
        ctx.save_for_backward(branch, None if y is None else residual, post, gate, pre, stats)
        ctx.rest = kinds, scale, residual_scale, s is not None, y is not None
        ctx.set_materialize_grads(False)
        return (s, y) if s is not None and y is not None else s if y is None else y

    @staticmethod
    @_once
    def backward(ctx, *grads):
        branch, residual, post, gate, pre, stats = ctx.saved_tensors
        if _capturing(ctx.rest[0][0]):
            raise RuntimeError("mi355moe: the backward pass of an eagerly recorded norm cannot be captured; capture "
                               "norm.join_forward and norm.join_backward")
        kinds, scale, residual_scale, has_s, has_y = ctx.rest
        return (*_backward(kinds, grads[0] if has_s else None, grads[-1] if has_y else None, stats, branch, residual, post, gate, pre,
                           scale, residual_scale, ctx.needs_input_grad), None, None, None, None, None)


def _call(branch, residual, post, gate, pre, eps, scale, residual_scale, need_s):
    kinds = _check(branch, residual, post, gate, pre)
    if torch.is_grad_enabled() and (branch.requires_grad or any(t is not None and t.requires_grad for t in (residual, post, gate, pre))):
        if _capturing(kinds[0]):
            raise RuntimeError("mi355moe: a norm cannot record a gradient during graph capture; capture norm.join_forward and "
                               "norm.join_backward")
        return _Join.apply(branch, residual, post, gate, pre, kinds, eps, scale, residual_scale, need_s)
    s, y, _ = _forward(kinds, branch, residual, post, gate, pre, eps, scale, residual_scale, need_s, False)
    return (s, y) if s is not None and y is not None else s if y is None else y


def join(branch: torch.Tensor, residual: torch.Tensor | None = None, post: torch.Tensor | None = None,
         gate: torch.Tensor | None = None, pre: torch.Tensor | None = None, eps: float = 1e-6, scale: float = 1.0,
         residual_scale: float = 1.0):
    """(s, y), or s without pre: a block's output `branch` [..., H] normed by post, times gate and scale, added to
    residual_scale * residual, and the sum normed by pre. residual is shaped and typed like branch; post and pre are [H] of one
    dtype; gate is [H], [..., 1] or [..., H] of any. Differentiable once in the five tensors by reverse mode (forward-mode
    derivatives are refused). While a graph is captured, a call that would record a gradient, and the backward pass of an
    eager one, are refused."""
    return _call(branch, residual, post, gate, pre, float(eps), float(scale), float(residual_scale), True)


def rms(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """x * r(x) * weight over the last dimension, with join's types and gradients."""
    if weight is None:
        raise ValueError("rms needs a weight")
    return _call(x, None, None, None, weight, float(eps), 1.0, 1.0, False)
