"""Each call of tests/path_cases.py launches the kernels it is there for: a changed rule shows here, and cannot leave a kernel
without its test unnoticed. No GPU needed."""
from __future__ import annotations

import pytest

import launches
import path_cases as cases

pytestmark = pytest.mark.skipif(not launches.compiler(), reason="no C compiler")


def _hold(calls, wants):
    for call, got, want in zip(calls, launches.launches(calls), wants):
        assert [k for k in got if k in want] == want, (call, got, want)
        kinds = ("mx_matmul", "mx_gateup", "mx_down", "gemm16", "gated_kernel", "gated_few", "join_kernel", "gated_join")
        assert not [k for k in got if k not in want and k.startswith(kinds)], (call, got, want)


def test_products():
    _hold([("matmul", c[:3]) for c in cases.PRODUCTS], [c[3] for c in cases.PRODUCTS])


def test_routed():
    calls, wants = [], []
    for c in cases.ROUTED:
        calls += [("moe", c[:5]), ("moe", (*c[:5], c[0] + 2))]
        wants += [c[6], c[6]]
    for c in cases.STORED:
        calls += [("moe", (*c[:5], 0, 0)), ("moe", c[:5])]
        wants += [c[5], c[5]]
    _hold(calls, wants)


def test_gated():
    calls, wants = [], []
    for fn, sizes in (("forward", cases.FORWARD), ("dx", cases.DX), ("dw", cases.DW)):
        for dt, code in (("bf16", "2"), ("fp16", "1")):
            calls += [(fn, (*c[:3], dt)) for c in sizes]
            wants += [[k.replace("<2", "<" + code) for k in c[4]] for c in sizes]
    _hold(calls, wants)


def test_every_kind_is_there():
    """The kernels of the library that multiply: each is some case's."""
    seen = {k for lst, at in ((cases.PRODUCTS, 3), (cases.ROUTED, 6), (cases.FORWARD, 4), (cases.DX, 4), (cases.DW, 4)) for c in lst for k in c[at]}
    made = launches.kernels()
    want = {k for k in made if k.startswith(("mx_matmul_", "mx_gateup_", "mx_down_"))}
    want |= {k for k in made if k.startswith(("gemm16_kernel<2", "gated_kernel<2", "gated_few_kernel<2", "gated_join_kernel<2"))}
    # (the direct path's gate/up kernel has a form for each type of x)
    missing = {k for k in want - seen if not k.startswith("mx_gateup_direct")}
    assert not missing, missing
