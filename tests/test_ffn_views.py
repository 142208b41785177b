"""The strides that the gated block's calls hand to the C entry points, for views that a user's program makes. No GPU needed:
the C layer takes strides of whole 16 bytes, at most 2^22 values for x."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("stride", [65, 100, 4099, (1 << 22) + 8, 8388608])
def test_one_row_has_no_stride(rows, stride):
    from mi355moe import ffn
    H = 64
    t = torch.empty_strided((rows, H), (stride, 1), dtype=torch.float16)
    r = ffn._rows16(t)
    assert r.shape == t.shape and ffn._row_stride(r) == H


@pytest.mark.parametrize("stride,kept", [(64, True), (72, True), (100, False), (1 << 22, True), ((1 << 22) + 8, False)])
def test_rows_are_copied_where_the_stride_does_not_do(stride, kept):
    from mi355moe import ffn
    base = torch.zeros(stride + 128, dtype=torch.float16)
    base = base[(-base.data_ptr() % 16) // 2:]
    t = base.as_strided((2, 64), (stride, 1))
    r = ffn._rows16(t)
    assert (r.data_ptr() == t.data_ptr()) == kept and ffn._row_stride(r) == (stride if kept else 64)
    assert ffn._row_stride(r) % 8 == 0 and ffn._row_stride(r) <= 1 << 22
