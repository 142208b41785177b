"""The far ends of the dense product's activations: where act(z) and act'(z) are small beside 1 they are held to their own size, not
to 1's.

z is exact (a row of one value times one weight of 1). Relative bounds, U half a step of fp32 at 1, before the result's own rounding:

  silu, gelu_tanh   e^-v carries U for each rounding of v, and of v times log2(e), times |v|, and the exponential's and the
                    reciprocal's steps; v is z, or 1.6 (z + 0.0447 z^3) in five roundings: (2 |z| + 16) U and (7 |v| + 16) U. The
                    slope s (1 + z (1 - s)) has |1 + z| for a factor, of which 1 - s takes a U: at most 2 |z| / |1 + z| U more.
  gelu              e^(-z^2 / 2) carries 3 (z^2 / 2) U likewise, the polynomial is within 2^-18 of erfc and its evaluation within 16 U;
                    the slope Phi + z phi adds two numbers that stand as 1 to z^2, so their errors grow by (z^2 + 1) / (z^2 - 1).

The ends are where the exponential or the reciprocal leaves fp32's normal numbers: z = -80 for silu, -12.5 for gelu, -9.5 for gelu_tanh."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

U = ref.U
ENDS = {"silu": (-80.0, -4.0), "gelu": (-12.5, -3.0), "gelu_tanh": (-9.5, -3.0)}


def _exact(name, z):
    """(act(z), act'(z), a relative bound of either) with nothing cancelled: math.erfc for Phi."""
    if name == "silu":
        s = 1.0 / (1.0 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s)), (2 * np.abs(z) + 16) * U + 2 * np.abs(z) / np.abs(1 + z) * U
    if name == "gelu":
        c = np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in z])
        slope = c + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        return z * c, slope, (1.5 * z * z * U + 2.0 ** -18 + 16 * U) * (z * z + 1) / (z * z - 1)
    a, b = 2 * math.sqrt(2 / math.pi), 0.044715
    v = a * (z + b * z ** 3)
    s = 1.0 / (1.0 + np.exp(-v))
    inner = z * (1 - s) * a * (1 + 3 * b * z * z)
    return z * s, s * (1 + inner), (7 * np.abs(v) + 16) * U + 8 * np.abs(inner) / np.abs(1 + inner) * U


@pytest.mark.parametrize("act", list(ENDS))
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_small_values(cuda, act, dt):
    from mi355moe import ffn
    lo, hi = ENDS[act]
    for rows in (40, 5000):                                      # by the streaming kernel, by tiles
        x = torch.linspace(lo, hi, rows, device="cuda").to(dt)[:, None].contiguous()
        one = torch.zeros(16, 1, device="cuda", dtype=dt)
        one[3] = 1.0
        y, z = ffn.linear_forward(x, one, activation=act, save=True)
        assert torch.equal(z[:, 3], x[:, 0].float())
        v = x[:, 0].double().cpu().numpy()
        want, _, tol = _exact(act, v)
        name = str(dt).replace("torch.", "")
        h, t = ref.HALF[name], ref.TINY[name]
        got = y[:, 3].double().cpu().numpy()
        bad = ~(np.abs(got - want) <= np.abs(want) * (tol * (1 + h) + h) + t)
        assert not bad.any(), (act, rows, v[bad][:4], got[bad][:4], want[bad][:4], int(bad.sum()))


@pytest.mark.parametrize("act", list(ENDS))
def test_small_slopes(cuda, act):
    """The bias' gradient of one row and dout = 1 is the slope in fp32."""
    from mi355moe import ffn
    lo, hi = ENDS[act]
    N = 4001
    z = torch.linspace(lo, hi, N, device="cuda")[None]
    x, w = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16), torch.ones(N, 8, device="cuda", dtype=torch.bfloat16)
    d = torch.ones(1, N, device="cuda", dtype=torch.bfloat16)
    got = ffn.linear_backward(d, z, x, w, act, torch.float32, need_dx=False, need_dw=False)[2].double().cpu().numpy()
    v = z[0].double().cpu().numpy()
    _, want, tol = _exact(act, v)
    bad = ~(np.abs(got - want) <= np.abs(want) * (tol + 8 * U))
    assert not bad.any(), (act, v[bad][:4], got[bad][:4], want[bad][:4], float(np.abs(got / want - 1).max()))
