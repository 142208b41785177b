"""Each call of tests/block_cases.py launches the kernels it is there for, every kernel of these operators is some case's, and a
launch that fails is reported by the call that made it. No GPU needed."""
from __future__ import annotations

import pytest

import block_cases as cases
import launches

pytestmark = pytest.mark.skipif(not launches.compiler(), reason="no C compiler")

CODES = {"bf16": "2", "fp16": "1", "fp32": "0"}


def _as(kernels, dt):
    return [k.replace("<2", "<" + CODES[dt], 1) for k in kernels]


def _calls():
    calls, wants = [], []
    for dt in ("bf16", "fp16"):
        for fn, sizes in (("linear", cases.LINEAR), ("dx", cases.DX), ("dw", cases.DW)):
            calls += [(fn, (*c[:3], dt)) for c in sizes]
            wants += [_as(c[3], dt) for c in sizes]
    for dt in ("bf16", "fp16", "fp32"):
        for c in cases.NORM:
            calls += [("norm", (*c[:2], dt)), ("norm_grad", (*c[:2], dt))]
            wants += [_as(c[2], dt), _as(c[3], dt)]
        for c in cases.ROWS:
            calls += [("back", (*c[:3], dt)), ("back_grad", (*c[:3], dt))]
            wants += [_as(c[4], dt), _as(c[5], dt)]
    for c in cases.ROWS:
        calls += [("to", (*c[:3], "bf16")), ("to", (*c[:3], "fp16"))]
        wants += [c[3], c[3]]
    calls += [("to", (40, 6, 72, "fp32")), ("to", (40, 6, 520, "fp32"))]
    wants += [["rows_scatter_kernel<4,0>"], ["rows_scatter_kernel<4,1>"]]
    for c in cases.SORT:
        for wide in (0, 1):
            calls.append(("sort", (*c[:3], wide)))
            wants.append(c[3])
    # what a gradient launches beside its products
    calls += [("grads", (70, 72, 40, "bf16")), ("grads", (70, 72, 40, "fp16")), ("grads", (70, 72, 40, "fp16", 1)), ("norm_grad", (9, 520, "bf16", 0))]
    small = [cases._tiles(1, 0, cases.S64), cases._tiles(1, 1, cases.S64)]
    wants += [["linear_dz_kernel<2>", "linear_dbias_kernel", *small],
              ["linear_top_kernel<1>", "linear_dz_kernel<1>", "linear_dbias_kernel", *_as(small, "fp16")],
              ["linear_dz_kernel<1>", "linear_dbias_kernel", *_as(small, "fp16")], ["norm_grad_kernel<2,1>"]]
    return calls, wants


def test_paths_and_failed_launches():
    calls, wants = _calls()
    (made, *got), silent = cases.run(calls)
    for call, g, w in zip(calls, got, wants):
        assert g == w, (call, g, w)
    assert not silent
    seen = {k for names in got for k in names}
    kinds = ("linear_", "norm_", "rows_", "sort_count", "sort_place")
    missing = {k for k in made if k.startswith(kinds)} - seen
    assert not missing, missing
