"""A kernel launch that fails is reported by the call that made it, whichever of its launches it is. No GPU needed."""
from __future__ import annotations

import pytest

import launches
import path_cases as cases


@pytest.mark.skipif(not launches.compiler(), reason="no C compiler")
def test_failed_launches_are_reported():
    calls = [("quant", (9, 64)), ("dequant", (9, 64)), ("arrange", (2, 5, 96)), ("matmul", (100, 70, 16544))]   # (arranged, in parts)
    calls += [("matmul", c[:3]) for c in cases.PRODUCTS] + [("moe", c[:5]) for c in cases.ROUTED]
    for dt in ("bf16", "fp16"):
        calls += [(fn, (*c[:3], dt)) for fn, sizes in (("forward", cases.FORWARD), ("dx", cases.DX), ("dw", cases.DW)) for c in sizes]
    assert not launches.silent_failures(calls)
