"""The largest sizes that the calls around a layer's experts take launch grids that the runtime takes: fewer than 2^32 threads a
dimension. On the host, with the launch functions replaced (tests/launches.py), where nothing of these sizes is allocated; and one
size beyond the first dimension on the GPU."""
from __future__ import annotations

import pytest

import block_cases as cases
import launches

LIMIT = "if ((unsigned long)gr.x * bl.x >> 32 || (unsigned long)gr.y * bl.y >> 32 || gr.y > 65535 || gr.z > 65535) return last = 9;"


@pytest.mark.skipif(not launches.compiler(), reason="no C compiler")
def test_largest_grids(monkeypatch):
    at = "if (!gr.x || !gr.y || !gr.z) return last = 9;"
    assert at in launches.STUB
    monkeypatch.setattr(launches, "STUB", launches.STUB.replace(at, at + " " + LIMIT))
    calls = []
    for H in (8, 64, 512, 1032, 2048, 4096, 65536):
        for T, k in ((1 << 24, 1), (1 << 21, 8), (1 << 19, 32)):
            calls += [(fn, (T, k, H, dt)) for fn in ("to", "back", "back_grad") for dt in ("bf16", "fp32")]
    for H in (1, 64, 65, 512, 513, 1024, 4096, 8192, 8193, 16384):
        calls += [(fn, (1 << 26, H, dt)) for fn in ("norm", "norm_grad") for dt in ("bf16", "fp32")]
    calls += [(fn, (M, K, N)) for fn in ("linear", "dx", "dw", "grads") for M, K, N in ((1 << 24, 8, 8), (1 << 24, 1027, 64), (8, 65536, 1 << 18),
                                                                                      (1 << 18, 64, 1 << 18))]
    calls += [("sort", (1 << 24, 1, 4096)), ("sort", (1 << 19, 32, 1))]
    (_, *got), silent = cases.run(calls)
    assert all(got) and not silent


@pytest.mark.gpu
def test_more_than_a_million_workgroups(cuda):
    """Beyond 2^20 workgroups the launches count on in a second dimension: the last tokens' rows are those of a short call."""
    import torch
    from mi355moe import dispatch, norm
    T, H = (1 << 20) + 5, 1032
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, H, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(T, 1, generator=g, device="cuda")
    ids = torch.randint(0, 3, (T, 1), generator=g, device="cuda")
    plan = dispatch.sort_tokens(ids, 2)
    at = plan.row[:, 0].long()
    live = at >= 0
    place = torch.where(live, at, ~at)
    rows = dispatch.to_experts(x, plan)
    out = dispatch.from_experts(rows, w, plan, x)
    drows, dw = dispatch.from_experts_backward(x, rows, w, plan)
    s, y, stats = norm.join_forward(x, x, pre=w[:H, 0])
    assert bool((s == (2 * x.float()).to(x.dtype)).all())
    for t in (slice(0, 64), slice(T // 2, T // 2 + 64), slice(T - 64, T)):
        kept = torch.where(live[t, None], x[t], torch.zeros_like(x[t]))
        assert torch.equal(rows[place[t]], kept)
        want = x[t].double() + w[t].double() * kept.double()
        assert float((out[t].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
        want = w[t].double() * kept.double()
        assert float((drows[place[t]].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
        want = (x[t].double() * kept.double()).sum(1)
        # (squares: a sum of 1032 of them in 5 steps a thread, 6 a wave, 5 over the waves, each within 2^-24 of itself)
        assert float((dw[t, 0].double() - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max())
        a, b, c = norm.join_forward(x[t].clone(), x[t].clone(), pre=w[:H, 0])
        assert torch.equal(s[t], a) and torch.equal(y[t], b) and torch.equal(stats[t], c)
