"""The gated block on views of one row: the last token of a prompt, a slice of a wider buffer, the gradient of a concatenation."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(T, H, I, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    w = (torch.randn(2 * I, H, generator=g, device="cuda") * 0.3).bfloat16()
    dh = torch.randn(T, I, generator=g, device="cuda").bfloat16()
    return x, w, dh


@pytest.mark.parametrize("T", [0, 1, 2])
@pytest.mark.parametrize("off", [0, 8])
def test_rows_of_a_wider_buffer(cuda, T, off):
    from mi355moe import ffn
    H, I = 64, 24
    x, w, dh = _inputs(T, H, I, 3)
    xb, db = torch.zeros(max(T, 1), 100, dtype=x.dtype, device="cuda"), torch.zeros(max(T, 1), 45, dtype=x.dtype, device="cuda")
    xb[:T, off:off + H], db[:T, off:off + I] = x, dh
    xv, dv = xb[:T, off:off + H], db[:T, off:off + I]
    h, gu = ffn.gated_forward(x, w, 2.0, save=True)
    hv, guv = ffn.gated_forward(xv, w, 2.0, save=True)
    assert torch.equal(h, hv) and torch.equal(gu, guv) and torch.equal(ffn.gated(xv, w, 2.0), h)
    for a, b in zip(ffn.gated_backward(dh, gu, x, w, 2.0), ffn.gated_backward(dv, gu, xv, w, 2.0)):
        assert torch.equal(a, b)


def test_last_token_of_a_prompt(cuda):
    """hidden[:, -1] of one sequence of 2048 tokens: a row whose stride is the whole sequence, 8388608 values."""
    from mi355moe import ffn
    H, I = 4096, 64
    hidden = torch.randn(1, 2048, H, device="cuda").bfloat16()
    _, w, _ = _inputs(1, H, I, 5)
    last = hidden[:, -1]
    assert last.stride(0) == 2048 * H
    assert torch.equal(ffn.gated(last, w, 10.0), ffn.gated(last.clone(memory_format=torch.contiguous_format), w, 10.0))


def test_gradient_of_a_concatenation(cuda):
    """The gradient that reaches one token's block is a slice of a wider one."""
    from mi355moe import ffn
    x, w, _ = _inputs(1, 64, 24, 7)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    extra = torch.ones(1, 13, dtype=x.dtype, device="cuda")
    c = torch.randn(1, 37, device="cuda").bfloat16()
    (torch.cat([ffn.gated(xr, wr, 2.0), extra], 1) * c).sum().backward()
    _, gu = ffn.gated_forward(x, w, 2.0, save=True)
    dx, dw = ffn.gated_backward(c[:, :24].clone(memory_format=torch.contiguous_format), gu, x, w, 2.0)
    assert torch.equal(xr.grad, dx) and torch.equal(wr.grad, dw)
