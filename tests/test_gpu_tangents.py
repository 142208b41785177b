"""Forward-mode derivatives of the gated block: refused, never dropped."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def test_gated_refuses_forward_mode(cuda):
    from mi355moe import ffn
    x, w = torch.randn(3, 64, device="cuda").half(), torch.randn(32, 64, device="cuda").half()
    want, gu = ffn.gated_forward(x, w, 2.0, save=True)
    dh = torch.ones_like(want)
    with fwd.dual_level():
        dx, dw, dd = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, dh))
        for args in ((dx, w), (x, dw), (dx.reshape(1, 3, 64), w), (dx.detach().requires_grad_(), dw)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ffn.gated(*args, 2.0)
            with pytest.raises(RuntimeError, match="forward-mode"):
                ffn.gated_forward(*args, 2.0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ffn.gated_backward(dd, gu, x, w, 2.0)
        assert torch.equal(ffn.gated(x, w, 2.0), want)
        assert torch.equal(ffn.gated(fwd.unpack_dual(dx).primal, w, 2.0), want)
