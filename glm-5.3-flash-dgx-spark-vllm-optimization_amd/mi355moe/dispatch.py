"""Tokens sorted by expert, and back with weights applied, with gradients.

For callers whose experts are not this package's (its own experts sort inside their calls): 16-bit experts that are tuned, or
an exchange between expert-parallel ranks.

    plan = sort_tokens(topk_ids, n)                                # rows, by expert; no host synchronisation
    rows = to_experts(x, plan)                                     # [T * topk, H]; expert e: plan.offsets[e] .. offsets[e + 1]
    out = from_experts(experts(rows), topk_weights, plan, shared)  # [T, H]: shared + the weighted rows of each token

  sort_tokens            the order: pairs by (local expert, pair index)
  to_experts             every pair's token row in that order, differentiable in x
  from_experts           the weighted sum per token in fp32, differentiable in rows, weights and shared
  from_experts_backward  its explicit gradients (for capture; to_experts' gradient is from_experts without weights)

Rows are fp32, fp16 or bf16. Every call runs on the current stream of its tensors' device; outputs and scratch come from torch's
caching allocator. No atomics on values: two calls give the same bits.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .ops import (_addr, _capturing, _current_device, _need_cuda, _no_tangents, _on_device, _once, _packed, _raw_stream, _rows_any,
                  _stream_at, ids_dtype_code, weight_dtype_code)


@functools.lru_cache(maxsize=4096)
def _sort_bytes(T: int, topk: int, n: int) -> int:
    return _lib.lib().mi355moe_sort_tokens_workspace_bytes(T, topk, n)


class SortedTokens:
    """The order of a router's picks, made by sort_tokens. row int32 [T, topk]: each pair's row, or ~row (negative) for a pair
    that no local expert takes (their rows come behind the others, and hold zeros); pair int32 [T * topk]: the pair of each
    row, or ~pair; offsets int32 [n + 1]: where each expert's rows begin, offsets[n] the number of rows that experts have."""

    __slots__ = ("_words", "tokens", "topk", "n")

    def __init__(self, words: torch.Tensor, tokens: int, topk: int, n: int):
        self._words, self.tokens, self.topk, self.n = words, tokens, topk, n      # row, pair, offsets, one behind the other

    @property
    def row(self) -> torch.Tensor:
        return self._words.as_strided((self.tokens, self.topk), (self.topk, 1))

    @property
    def pair(self) -> torch.Tensor:
        P = self.tokens * self.topk
        return self._words.as_strided((P,), (1,), P)

    @property
    def offsets(self) -> torch.Tensor:
        return self._words.as_strided((self.n + 1,), (1,), 2 * self.tokens * self.topk)

    @property
    def device(self) -> torch.device:
        return self._words.device


def sort_tokens(topk_ids: torch.Tensor, n: int, expert_map: torch.Tensor | None = None) -> SortedTokens:
    """The pairs of topk_ids [T, topk] (int32 or int64) in the order (local expert, pair index). Without expert_map an id in [0,
    n) is its local expert; with it ([ids] of global id -> local id) an id's entry is. Every other pair is dropped: it is no
    expert's, its row comes behind offsets[n]."""
    dev = _need_cuda(topk_ids, expert_map)
    code = ids_dtype_code(topk_ids.dtype)
    if topk_ids.dim() != 2 or topk_ids.shape[1] == 0:
        raise ValueError(f"topk_ids must be [T, topk], got {tuple(topk_ids.shape)}")
    if expert_map is not None:
        kind = expert_map.dtype
        if expert_map.dim() != 1 or kind.is_floating_point or kind.is_complex or kind == torch.bool:
            raise ValueError(f"expert_map must be a vector of whole numbers, got {kind} {tuple(expert_map.shape)}")
    T, topk = topk_ids.shape
    n, P = int(n), T * topk
    nb = _sort_bytes(T, topk, n)
    with _on_device(dev):
        ids = topk_ids.contiguous()
        em, n_global = None, 0
        if expert_map is not None:
            em = expert_map.to(torch.int64).contiguous()
            n_global = em.numel()
            if n_global == 0:
                em = ids.new_zeros(1, dtype=torch.int64)         # (no id has an entry; the address only says that there is a map)
        # the scratch lies behind the three tables (sizes that the library refuses: nothing to write)
        words = ids.new_empty(2 * P + n + 1 + nb // 4 if nb >= 0 else 1, dtype=torch.int32)
        at = words.data_ptr()
        _lib.check("mi355moe_sort_tokens", _lib.lib().mi355moe_sort_tokens(
            _addr(ids), code, T, topk, _addr(em), n_global, n, at, at + 4 * P, at + 8 * P, at + 4 * (2 * P + n + 1) if nb > 0 else None,
            max(nb, 0), _raw_stream(dev)))
    return SortedTokens(words, T, topk, n)


def _check(plan: SortedTokens, what: str, t: torch.Tensor, rows: int, dev: torch.device) -> int:
    code = weight_dtype_code(t.dtype)
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] == 0:
        raise ValueError(f"{what} must be [{rows}, H], got {tuple(t.shape)}")
    if plan.device != dev:
        raise ValueError(f"the order is on {plan.device}, {what} on {dev}")
    return code


def _to_experts(x: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    dev = _need_cuda(x)
    return _scatter(dev, _check(plan, "x", x, plan.tokens, dev), x, plan)


def _scatter(dev, code, x, plan):
    """_to_experts of arguments that have been looked at."""
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _scatter(dev, code, x, plan)
    T, topk, H = plan.tokens, plan.topk, x.shape[1]
    x, ldx = (x, H) if x.is_contiguous() else _rows_any(x)
    rows = x.new_empty(T * topk, H)
    rc = _lib.lib().mi355moe_rows_to_experts(x.data_ptr(), code, T, H, ldx, plan._words.data_ptr(), topk, rows.data_ptr(),
                                               _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_rows_to_experts", rc)
    return rows


def _check_back(rows, weights, plan, shared):
    dev = _need_cuda(rows, weights, shared)
    code = _check(plan, "rows", rows, plan.tokens * plan.topk, dev)
    if weights is not None and weights.shape != (plan.tokens, plan.topk):
        raise ValueError(f"weights must be {(plan.tokens, plan.topk)}, got {tuple(weights.shape)}")
    if shared is not None and (shared.dtype != rows.dtype or shared.shape != (plan.tokens, rows.shape[1])):
        raise ValueError(f"shared must be {rows.dtype} {(plan.tokens, rows.shape[1])}, got {shared.dtype} {tuple(shared.shape)}")
    return dev, code


def _from_experts(rows, weights, plan, shared):
    dev, code = _check_back(rows, weights, plan, shared)
    return _gather(dev, code, rows, weights, plan, shared)


def _gather(dev, code, rows, weights, plan, shared):
    """_from_experts of arguments that have been looked at."""
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _gather(dev, code, rows, weights, plan, shared)
    wcode = _lib.F32 if weights is None else weight_dtype_code(weights.dtype)
    T, H = plan.tokens, rows.shape[1]
    rows = rows if rows.is_contiguous() else _packed(rows)
    weights = weights if weights is None or weights.is_contiguous() else _packed(weights)
    shared, lds = (shared, H) if shared is None or shared.is_contiguous() else _rows_any(shared)
    out = rows.new_empty(T, H)
    rc = _lib.lib().mi355moe_rows_from_experts(
        rows.data_ptr(), code, T, H, plan._words.data_ptr(), plan.topk, weights if weights is None else weights.data_ptr(), wcode,
        shared if shared is None else shared.data_ptr(), lds, out.data_ptr(), H, _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_rows_from_experts", rc)
    return out


def from_experts_backward(dout: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, plan: SortedTokens, need_rows: bool = True,
                          need_weights: bool = True):
    """(drows, dweights), None where not needed, of from_experts(rows, weights, plan) from dout [T, H]: drows in rows' dtype, zero
    behind offsets[n]; dweights in weights' dtype, zero for the pairs that no local expert takes. shared's gradient is dout. rows'
    values are read for dweights only. (Without weights, rows' gradient is to_experts(dout, plan).)"""
    if weights is None:
        raise ValueError("from_experts_backward needs weights; without them the gradient of rows is to_experts(dout, plan)")
    dev, code = _check_back(rows, weights, plan, None)
    _need_cuda(rows, dout)
    _no_tangents("from_experts_backward", dout, rows, weights)
    H = rows.shape[1]
    if dout.dtype != rows.dtype or dout.shape != (plan.tokens, H):
        raise ValueError(f"dout must be {rows.dtype} {(plan.tokens, H)}, got {dout.dtype} {tuple(dout.shape)}")
    return _from_grads(dev, code, dout, rows, weights, plan, need_rows, need_weights)


def _from_grads(dev, code, dout, rows, weights, plan, need_rows, need_weights):
    """from_experts_backward of arguments that have been looked at. rows may be None where dweights is not needed."""
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return _from_grads(dev, code, dout, rows, weights, plan, need_rows, need_weights)
    H = dout.shape[1]
    dout, ldd = (dout, H) if dout.is_contiguous() else _rows_any(dout)
    weights = weights if weights.is_contiguous() else _packed(weights)
    drows = dw = None
    if need_rows:
        drows = torch.empty_like(rows) if rows is not None and rows.is_contiguous() else dout.new_empty(plan.tokens * plan.topk, H)
    if need_weights:
        dw = torch.empty_like(weights)
        rows = rows if rows.is_contiguous() else _packed(rows)
    rc = _lib.lib().mi355moe_rows_from_experts_backward(
        dout.data_ptr(), code, plan.tokens, H, ldd, plan._words.data_ptr(), plan.topk, weights.data_ptr(), weight_dtype_code(weights.dtype),
        rows.data_ptr() if need_weights else None, drows if drows is None else drows.data_ptr(), dw if dw is None else dw.data_ptr(),
        _stream_at(dev.index))
    if rc:
        _lib.check("mi355moe_rows_from_experts_backward", rc)
    return drows, dw


_NOT_CAPTURED = ("mi355moe: {} cannot {} during graph capture; capture it under torch.no_grad with its explicit gradient "
                 "(from_experts without weights, from_experts_backward)")


# (autograd gives a backward pass gradients of the outputs' shapes and types: they are not looked at again)
class _To(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        dev = _need_cuda(x)
        ctx.rest = dev, _check(plan, "x", x, plan.tokens, dev), plan
        return _scatter(dev, ctx.rest[1], x, plan)

    @staticmethod
    @_once
    def backward(ctx, drows):
        dev, code, plan = ctx.rest
        if _capturing(dev):
            raise RuntimeError(_NOT_CAPTURED.format("to_experts", "run an eager call's backward pass"))
        return _gather(dev, code, drows, None, plan, None), None


class _From(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan, shared):
        dev, code = _check_back(rows, weights, plan, shared)
        ctx.rest = dev, code, plan
        # (rows are read for the weights' gradient only: kept for nothing else, [T * topk, H] would stay until the backward pass)
        need = ctx.needs_input_grad
        ctx.save_for_backward(rows if need[1] else None, weights if need[0] or need[1] else None)
        return _gather(dev, code, rows, weights, plan, shared)

    @staticmethod
    @_once
    def backward(ctx, dout):
        dev, code, plan = ctx.rest
        if _capturing(dev):
            raise RuntimeError(_NOT_CAPTURED.format("from_experts", "run an eager call's backward pass"))
        rows, weights = ctx.saved_tensors
        need = ctx.needs_input_grad
        drows = dw = None
        if weights is None:
            drows = _scatter(dev, code, dout, plan) if need[0] else None
        elif need[0] or need[1]:
            drows, dw = _from_grads(dev, code, dout, rows, weights, plan, need[0], need[1])
        return drows, dw, None, dout if need[3] else None


def _records(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def to_experts(x: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    """rows [T * topk, H] of x [T, H]: row plan.row[t, j] is x[t]; the rows behind plan.offsets[n] are zero. Differentiable once in
    x by reverse mode (forward-mode derivatives are refused). A call that would record a gradient, and the backward pass of an
    eager one, are refused while a graph is captured."""
    _no_tangents("to_experts", x)
    if _records(x):
        if _capturing(x.device):
            raise RuntimeError(_NOT_CAPTURED.format("to_experts", "record a gradient"))
        return _To.apply(x, plan)
    return _to_experts(x, plan)


def from_experts(rows: torch.Tensor, weights: torch.Tensor | None, plan: SortedTokens,
                 shared: torch.Tensor | None = None) -> torch.Tensor:
    """out [T, H] = shared + the sum over j of weights[t, j] * rows[plan.row[t, j]] (weights None: ones), j ascending, in fp32 with
    one rounding to rows' dtype. Pairs that no local expert takes count as nothing, whatever their weight. Differentiable once
    in rows, weights and shared, with the limits of to_experts."""
    _no_tangents("from_experts", rows, weights, shared)
    if _records(rows, weights, shared):
        if _capturing(rows.device):
            raise RuntimeError(_NOT_CAPTURED.format("from_experts", "record a gradient"))
        return _From.apply(rows, weights, plan, shared)
    return _from_experts(rows, weights, plan, shared)
