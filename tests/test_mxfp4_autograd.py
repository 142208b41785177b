"""What the MXFP4 calls do with tensors that autograd follows: a gradient is refused or raises, never lost. No GPU needed."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_outputs_that_autograd_follows():
    from mi355moe.mxfp4 import _may_write
    plain, leaf = torch.zeros(2, 3), torch.zeros(2, 3, requires_grad=True)
    result = leaf * 2
    for adds in (False, True):
        _may_write(plain, "call", adds, plain)
        for out, inputs in ((leaf, ()), (leaf[:1], ()), (plain, (leaf,)), (plain, (plain, leaf)), (result, (result,))):
            with pytest.raises(RuntimeError, match="gradient"):
                _may_write(out, "call", adds, *inputs)
            with torch.no_grad():
                _may_write(out, "call", adds, *inputs)
    _may_write(result, "call", True, plain)
    _may_write(result[:, 1:], "call", True, plain)
    with pytest.raises(RuntimeError, match="gradient"):
        _may_write(result, "call", False, plain)
    with fwd.dual_level():
        d = fwd.make_dual(plain, plain)
        for out, inputs in ((d, ()), (plain, (d,))):
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                _may_write(out, "call", True, *inputs)


def test_results_of_inputs_that_need_gradients():
    from mi355moe.mxfp4 import _without_gradient
    out, x, w = torch.ones(2, 3), torch.zeros(2, 4), torch.zeros(2, 1)
    assert _without_gradient(out, "call", x, w) is out
    for a, b in ((x.clone().requires_grad_(), w), (x, w.clone().requires_grad_())):
        r = _without_gradient(out, "call", a, b)
        assert r.requires_grad and torch.equal(r, out)
        with pytest.raises(RuntimeError, match="no gradient"):
            r.sum().backward()
        with torch.no_grad():
            assert _without_gradient(out, "call", a, b) is out
