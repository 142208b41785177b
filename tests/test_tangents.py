"""Tensors that carry a forward-mode derivative are refused: nothing on the host would otherwise notice that the kernels lose
it. No GPU needed."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_tangents_are_refused():
    from mi355moe import ops
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    ops._no_tangents("x", x, None, w)
    with fwd.dual_level():
        ops._no_tangents("x", x, None, w)
        d = fwd.make_dual(x, torch.ones_like(x))
        for ts in ((d,), (w, d), (None, d[:1])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops._no_tangents("x", *ts)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                ops._no_tangents("x", *ts)
        ops._no_tangents("x", fwd.unpack_dual(d).primal, d.detach())
    ops._no_tangents("x", x)
