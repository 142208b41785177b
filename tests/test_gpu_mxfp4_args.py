"""Arguments that a call over the MXFP4 experts must not take for others."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_expert_map_without_entries(cuda):
    """No entry maps no id to an expert: refused, since an empty tensor's address says that there is no map."""
    from mi355moe import mxfp4
    ex = mxfp4.Mxfp4Experts.from_dense(torch.randn(2, 64, 64, device="cuda"), torch.randn(2, 64, 32, device="cuda"))
    x, ids, w = torch.randn(3, 64, device="cuda"), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, 1, device="cuda")
    with pytest.raises(ValueError, match="no entries"):
        mxfp4.moe_forward_ids(ex, x, ids, w, expert_map=torch.empty(0, dtype=torch.int64, device="cuda"))
    none = mxfp4.moe_forward_ids(ex, x, ids, w, expert_map=torch.full((1,), -1, device="cuda"))
    assert (none == 0).all()
