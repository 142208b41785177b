"""The operators around a layer's experts run together, as a layer has them: the norm before the block, the shared expert (gated
block and down projection), the tokens to their experts and back onto the shared expert's output, then the norm after the
block with its gate and residual sum and the norm before the next one. Forward and all gradients against float64 autograd."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gated64(x, w13, L):
    g, u = (x @ w13.t()).chunk(2, -1)
    g, u = g.clamp(max=L), u.clamp(-L, L)
    return g * torch.sigmoid(g) * u


def _rms64(v, w, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w


@pytest.mark.parametrize("T", [1, 7, 90])
def test_layer(cuda, T):
    from mi355moe import dispatch, ffn, norm
    n, topk, H, I, L, eps, dt = 6, 3, 136, 72, 10.0, 1e-5, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(T)
    new = lambda *s, f=1.0: torch.randn(*s, generator=g, device="cuda") * f  # noqa: E731
    leaf = {"x": new(T, H).to(dt), "pre": 1 + new(H, f=0.2), "s13": new(2 * I, H, f=0.15).to(dt), "s2": new(H, I, f=0.15).to(dt),
            "b2": new(H, f=0.2), "e13": new(n, 2 * I, H, f=0.15).to(dt), "e2": new(n, H, I, f=0.15).to(dt), "wts": torch.rand(T, topk, generator=g, device="cuda"),
            "post": 1 + new(H, f=0.2), "gate": new(H, f=0.5).to(dt), "next": 1 + new(H, f=0.2)}
    ids = torch.topk(torch.rand(T, n + 1, generator=g, device="cuda"), topk, dim=1).indices      # expert n is another rank's
    ds, dy = new(T, H).to(dt), new(T, H).to(dt)
    for v in leaf.values():
        v.requires_grad_()
    p = leaf
    x = norm.rms(p["x"], p["pre"], eps)
    shared = ffn.linear(ffn.gated(x, p["s13"], L), p["s2"], bias=p["b2"])
    plan = dispatch.sort_tokens(ids, n)
    rows = dispatch.to_experts(x, plan)
    at = plan.offsets.tolist()
    parts = [ffn.linear(ffn.gated(rows[a:b], w13, L), w2) for a, b, w13, w2 in zip(at, at[1:], p["e13"], p["e2"])]
    out = dispatch.from_experts(torch.cat([*parts, rows[at[-1]:]]), p["wts"], plan, shared=shared)
    s, y = norm.join(out, p["x"], post=p["post"], gate=p["gate"], pre=p["next"], eps=eps, scale=0.5, residual_scale=1.25)
    grads = torch.autograd.grad((s, y), list(p.values()), (ds, dy))

    q = {k: v.detach().double().requires_grad_() for k, v in leaf.items()}
    x = _rms64(q["x"], q["pre"], eps)
    total = _gated64(x, q["s13"], L) @ q["s2"].t() + q["b2"]
    for e in range(n):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        total = total.index_add(0, t, _gated64(x[t], q["e13"][e], L) @ q["e2"][e].t() * q["wts"][t, j, None])
    s64 = 1.25 * q["x"] + 0.5 * q["gate"] * _rms64(total, q["post"], eps)
    y64 = _rms64(s64, q["next"], eps)
    want = torch.autograd.grad((s64, y64), list(q.values()), (ds.double(), dy.double()))

    # bf16 rounds x, h, the shared and the routed output, [dg | du], dz and each gradient handed on: at most ten half steps of 2^-8
    # on a path, each relative to its own tensor; the norms' and the SwiGLU's slopes amplify by less than four
    tol = 10 * 2.0 ** -8 * 4
    for k, got, ref in (("s", s, s64), ("y", y, y64), *zip((f"d{k}" for k in p), grads, want)):
        assert torch.isfinite(got).all(), k
        assert float((got.double() - ref).norm()) <= tol * float(ref.norm()) + 1e-12, (k, float((got.double() - ref).norm()), float(ref.norm()))
