"""Sums over many rows: the gradients of weights, with inputs for which a row that is lost, or read in another's place, shows.

Bounds that grow with the rows hide single ones, so what is added up here is exact, or is zero but for a few rows:

  products   dout is +-1 in a few hundred rows and x is -1, 0 or 1, so that dW is a whole number of at most 8 bits
  norms      ds and dy are zero but in a few rows: those rows alone are in the bound"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block as ref

NAMES = ("branch", "residual", "post", "gate", "pre")


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


# ---------------------------------------------------------------------------------------------- the dense product


def _marks(M, row_bytes):
    """Rows at both ends of M, around every place where a power of two from 2^31 on divides the rows' bytes, and around the first
    and last rows of the parts that a contraction may be cut into: 240 at most, in order."""
    at = {*range(20), *range(M - 20, M)}
    for k in (31, 32, 33):
        r = (1 << k) // row_bytes
        at |= {i for i in range(r - 8, r + 9) if 0 <= i < M}
    for parts in (2, 4, 8, 16):
        for i in range(1, parts):
            at |= {M * i // parts, -(-M // 64 // parts) * 64 * i}
    at = sorted(i for i in at if 0 <= i < M)
    assert 60 <= len(at) <= 240
    return torch.tensor(at)


def _whole(M, K, N, at, device):
    """(x, dout) in bf16, and dW and the bias' gradient that they have, exactly."""
    g = torch.Generator(device=device).manual_seed(2)
    x = torch.randint(-1, 2, (M, K), generator=g, device=device, dtype=torch.int8).to(torch.bfloat16)
    d = torch.zeros(M, N, device=device, dtype=torch.bfloat16)
    signs = (torch.randint(0, 2, (len(at), N), generator=g, device=device) * 2 - 1).double()
    d[at.to(device)] = signs.to(torch.bfloat16)
    return x, d, signs.t().contiguous() @ x[at.to(device)].double(), signs.sum(0)


def test_a_lost_row_shows():
    """On the host: each of the rows changes every bias sum by 1, and dW in two of three columns; an exact comparison sees it."""
    M, K, N = 5000, 40, 24
    at = torch.tensor(sorted({*range(60), *range(2000, 2060), *range(M - 60, M)}))
    x, d, dw, db = _whole(M, K, N, at, "cpu")
    assert torch.equal(d.double().t() @ x.double(), dw) and dw.abs().max() <= 256 and torch.equal(dw.to(torch.bfloat16).double(), dw)
    for r in at.tolist():
        lost = d.clone()
        lost[r] = 0
        assert not torch.equal(lost.double().t() @ x.double(), dw) and not torch.equal(lost.double().sum(0), db)
    moved = x.roll(1, 0)                                          # every row's neighbour read in its place
    assert not torch.equal(d.double().t() @ moved.double(), dw)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [((1 << 21) + 3, 1032, 24), ((1 << 21) + 3, 24, 1032), ((1 << 17) + 5, 520, 264), (70001, 131, 40)])
def test_weights_of_long_contractions(cuda, M, K, N):
    """dW and the bias' gradient over rows of x, or of dout, whose bytes pass 32 bits, and over parts of the contraction."""
    from mi355moe import ffn
    at = _marks(M, 2 * max(K, N))
    x, d, dw, db = _whole(M, K, N, at, "cuda")
    w = torch.randn(N, K, device="cuda").to(torch.bfloat16)
    _, got, sums = ffn.linear_backward(d, None, x, w, None, torch.float32, need_dx=False)
    assert torch.equal(sums.double(), db), (sums.double() - db).abs().max()
    assert torch.equal(got.double(), dw), (got.double() - dw).abs().max()
    # and with every row's part in sums below 2^24, which fp32 has exactly in any order: dW rounded once
    d = torch.randint(-1, 2, (M, N), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    _, got, sums = ffn.linear_backward(d, None, x, w, None, torch.float32, need_dx=False)
    want = torch.zeros(N, K, device="cuda", dtype=torch.float64)
    for i in range(0, M, 1 << 18):
        want += d[i:i + (1 << 18)].double().t().contiguous() @ x[i:i + (1 << 18)].double()
    assert torch.equal(sums.double(), d.double().sum(0)) and torch.equal(got, want.to(torch.bfloat16))


# ---------------------------------------------------------------------------------------------- the norms


def _norm_case(R, H, gate, dt, rows, device, seed):
    """The five inputs, and ds and dy that are zero but in `rows`."""
    g = torch.Generator(device=device).manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    t = [(new(R, H) * 0.7 + 0.1).to(dt), (new(R, H) * 3).to(dt), 1 + 0.3 * new(H),
         new(*{"channel": (H,), "token": (R, 1), "full": (R, H)}[gate]), 1 + 0.3 * new(H)]
    d = []
    for _ in range(2):
        v = torch.zeros(R, H, device=device, dtype=dt)
        v[rows] = new(len(rows), H).to(dt)
        d.append(v)
    return t, d


def _norm_sums(t, d, rows):
    """{name: (gradient, bound)} of the sums over the rows: (256 + rows) U of the magnitude, of the rows that are not zero."""
    pick = [v if v.dim() == 1 else v[rows] for v in t]
    want = ref.norm_grads(*(_f64(v[rows]) for v in d), *(_f64(v) for v in pick), 1e-5, 0.5, 1.25)
    return {k: (want[k][0], (256 + len(rows)) * ref.U * want[k][1]) for k in NAMES if want[k][0].ndim == 1}


def _norm_rows(R, steps):
    """The first and last rows, and those around every place where a workgroup begins its next ones."""
    at = {0, 1, R - 1, R - 2, R // 2}
    for s in steps:
        at |= {i for i in (s - 1, s, s + 1) if 0 <= i < R}
    return sorted(at)


def test_a_lost_row_of_a_norm_shows():
    """On the host: without any one of the rows each sum is out of its bound, in most of its columns."""
    R, H = 700, 33
    rows = _norm_rows(R, (256, 512))
    for gate in ("channel", "token", "full"):
        t, d = _norm_case(R, H, gate, torch.float32, rows, "cpu", 1)
        want = _norm_sums(t, d, rows)
        for r in rows:
            lost = _norm_sums(t, d, [i for i in rows if i != r])
            for k, (v, tol) in want.items():
                # (the result's own rounding, at most bf16's, is in the comparison)
                assert (np.abs(lost[k][0] - v) > tol * 1.01 + 2.0 ** -8 * np.abs(v)).mean() > 0.5, (gate, r, k)


# rows, values, and how many rows the gradient has at once (1024 workgroups of 8 to 64 lanes a row; beyond 512 values a workgroup a row)
STEPS = [(40007, 33, 32 * 1024), (20003, 100, 16 * 1024), (9001, 200, 8 * 1024), (5003, 300, 4 * 1024), (4500, 520, 2048), (3001, 1032, 1280), (1100, 4099, 256),
         (700, 8200, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("R,H,step", STEPS)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_weights_of_many_rows(cuda, R, H, step, dt):
    """dpost, dpre and a channel's gate over more rows than the gradient has at once, the last workgroup part full."""
    from mi355moe import norm
    rows = _norm_rows(R, [k * step for k in range(1, R // step + 1)])
    assert R % 32 and len(rows) < 40
    for gate in ("channel", "token", "full"):
        t, d = _norm_case(R, H, gate, dt, rows, "cuda", R)
        _, _, stats = norm.join_forward(*t, 1e-5, 0.5, 1.25)
        got = dict(zip(NAMES, norm.join_backward(*d, stats, *t, 0.5, 1.25)))
        for k, (v, tol) in _norm_sums(t, d, rows).items():
            bad = ~(np.abs(_f64(got[k]) - v) <= tol + ref.U * np.abs(v))
            assert not bad.any(), (gate, k, np.argwhere(bad)[:5], int(bad.sum()))
        # rows without a gradient have none, the others theirs
        some = torch.zeros(R, dtype=torch.bool, device="cuda")
        some[rows] = True
        for k in ("branch", "residual"):
            assert torch.equal(got[k].abs().amax(1) > 0, some), (gate, k)
