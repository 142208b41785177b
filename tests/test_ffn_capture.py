"""The backward pass of an eager ffn.gated while a graph is captured: refused before anything is launched. On the host alone
(the capture is pretended), since what such a capture would record is not a thing to try on a GPU."""
from __future__ import annotations

import types

import pytest
import torch


def test_backward_is_refused_during_capture(monkeypatch):
    from mi355moe import ffn

    def launched(*a, **k):
        raise AssertionError("launched")

    monkeypatch.setattr(ffn, "gated_backward", launched)
    t = torch.zeros(2, 16)
    ctx = types.SimpleNamespace(saved_tensors=(t, t, t), limit=1.0, needs_input_grad=(True, True, False))
    monkeypatch.setattr(ffn, "_capturing", lambda dev: True)
    with pytest.raises(RuntimeError, match="captured"):
        ffn._Gated.backward(ctx, t)
    monkeypatch.setattr(ffn, "_capturing", lambda dev: False)
    with pytest.raises(AssertionError, match="launched"):
        ffn._Gated.backward(ctx, t)
