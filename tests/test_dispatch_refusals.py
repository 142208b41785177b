"""Arguments of the calls between a router and its experts that are refused by name."""
from __future__ import annotations

import pytest
import torch


def test_gradients_of_rows_back_need_weights():
    from mi355moe import dispatch
    plan = dispatch.SortedTokens(torch.zeros(16, dtype=torch.int32), 2, 2, 4)
    for need in ((True, True), (True, False), (False, True)):
        with pytest.raises(ValueError, match="needs weights"):
            dispatch.from_experts_backward(torch.zeros(2, 8), torch.zeros(4, 8), None, plan, *need)


@pytest.mark.gpu
def test_maps_of_complex_numbers(cuda):
    from mi355moe import dispatch
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for dt in (torch.complex64, torch.complex128):
        with pytest.raises(ValueError, match="whole numbers"):
            dispatch.sort_tokens(ids, 4, expert_map=torch.zeros(4, dtype=dt, device="cuda"))
