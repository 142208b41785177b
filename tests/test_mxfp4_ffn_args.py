"""Refusals of the MXFP4 and gated-block entry points: the C ABI's argument checks, which come before any launch (made-up
addresses are never read), the Python layer's, and the float64 definitions on known values. No GPU needed."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

P, NUL = ctypes.c_void_p(0x10000), ctypes.c_void_p(0)
ODD = ctypes.c_void_p(0x10001)
EINVAL, ESHAPE, ELIMIT, EWORKSPACE, EDTYPE = 1, 2, 3, 4, 5
F32, F16, BF16, I32, I64 = range(5)


@pytest.fixture(scope="module")
def L():
    from mi355moe import _lib
    return _lib.lib()


def test_quant_refusals(L):
    f = L.mi355moe_mxfp4_quant_rows
    assert f(P, I32, 1, 32, 32, P, P, NUL) == EDTYPE
    assert f(P, F32, -1, 32, 32, P, P, NUL) == ESHAPE
    assert f(P, F32, 1, 0, 32, P, P, NUL) == ESHAPE
    assert f(P, F32, 2, 32, 31, P, P, NUL) == ESHAPE
    assert f(P, F32, 1 << 40, 32, 32, P, P, NUL) == ELIMIT
    for a in ((NUL, P, P), (P, NUL, P), (P, P, NUL)):
        assert f(a[0], F32, 1, 32, 32, a[1], a[2], NUL) == EINVAL
    assert f(NUL, F32, 0, 32, 32, NUL, NUL, NUL) == 0
    g = L.mi355moe_mxfp4_dequant_rows
    assert g(P, P, 1, 32, P, I64, NUL) == EDTYPE
    assert g(P, P, 1, 0, P, F32, NUL) == ESHAPE
    assert g(P, NUL, 1, 32, P, F32, NUL) == EINVAL
    assert g(NUL, NUL, 0, 32, NUL, F32, NUL) == 0


def test_matmul_refusals(L):
    f, size = L.mi355moe_mxfp4_matmul, L.mi355moe_mxfp4_matmul_workspace_bytes
    ok = dict(a=P, sa=P, M=4, w=P, sw=P, N=8, K=64, out=P, dt=BF16, st=8, ws=P, nb=1 << 30)

    def call(**kw):
        d = {**ok, **kw}
        return f(d["a"], d["sa"], d["M"], d["w"], d["sw"], d["N"], d["K"], d["out"], d["dt"], d["st"], d["ws"], d["nb"], NUL)

    for K in (0, 16, 33, 48):
        assert call(K=K) == ESHAPE and size(4, 8, K) == -1
    assert call(N=0) == ESHAPE and call(M=-1) == ESHAPE and call(st=7) == ESHAPE
    assert call(M=(1 << 20) + 1) == ELIMIT and call(K=1 << 17) == ELIMIT
    assert call(dt=I32) == EDTYPE
    for k in ("a", "sa", "w", "sw", "out"):
        assert call(**{k: NUL}) == EINVAL
    assert call(a=ODD) == EINVAL and call(w=ODD) == EINVAL and call(K=128, sa=ODD) == EINVAL
    big = dict(M=4096, N=1024, K=160, st=1024)             # scales of no whole dwords, large tiles: arranged in the workspace
    assert call(**big, ws=ODD) == EINVAL
    assert size(4096, 1024, 160) > 0 and call(**big, ws=NUL) == EINVAL and call(**big, nb=size(4096, 1024, 160) - 1) == EWORKSPACE
    assert size(4, 8, 64) == 0 and size(100, 8, 160) == 0
    assert size(4, 8, 128) == 0
    assert call(M=0, a=NUL, out=NUL) == 0


def _layer(**kw):
    from mi355moe import _lib
    d = _lib.Mxfp4LayerDesc()
    d.n, d.hidden, d.intermediate, d.arranged = 8, 128, 128, 1
    for k in ("w13", "w13_scale", "w2", "w2_scale"):
        setattr(d, k, P)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_moe_refusals(L):
    f, size = L.mi355moe_mxfp4_moe_forward_ids, L.mi355moe_mxfp4_moe_workspace_bytes

    def call(layer=None, x=P, dt=BF16, xs=128, T=4, idt=I32, wdt=F32, topk=2, odt=BF16, os=128, opt=0, ws=P, nb=1 << 40, ng=0,
             em=NUL, lim=10.0):
        return f(ctypes.byref(layer or _layer()), x, dt, xs, T, P, idt, P, wdt, topk, em, ng, lim, P, odt, os, opt, ws, nb, NUL)

    assert call(_layer(n=0)) == ELIMIT and call(_layer(n=5000)) == ELIMIT
    assert call(_layer(hidden=48)) == ESHAPE and call(_layer(intermediate=0)) == ESHAPE
    assert call(_layer(hidden=32768)) == ELIMIT and call(_layer(arranged=2)) == EINVAL
    assert call(_layer(hidden=96, arranged=0)) == ESHAPE and call(_layer(intermediate=160, arranged=0)) == ESHAPE
    assert call(_layer(w13=NUL)) == EINVAL and call(_layer(w2=ODD)) == EINVAL and call(_layer(w2_scale=ODD)) == EINVAL
    assert call(x=NUL) == EINVAL and call(ws=NUL) == EINVAL and call(opt=2) == EINVAL and call(em=P, ng=-1) == EINVAL
    assert call(lim=-1.0) == EINVAL and call(lim=float("nan")) == EINVAL and call(ws=ODD) == EINVAL
    assert call(dt=I32) == EDTYPE and call(idt=F32) == EDTYPE and call(wdt=I64) == EDTYPE and call(odt=7) == EDTYPE
    assert call(xs=127) == ESHAPE and call(os=100) == ESHAPE
    assert call(topk=0) == ELIMIT and call(topk=33) == ELIMIT and call(T=40000) == ELIMIT
    lay = _layer()
    assert call(nb=size(ctypes.byref(lay), 4, 2) - 1) == EWORKSPACE
    assert size(ctypes.byref(_layer(hidden=48)), 4, 2) == -1 and size(ctypes.byref(lay), 4, 0) == -1
    assert call(T=0) == 0


def test_arrange_refusals(L):
    f, size = L.mi355moe_mxfp4_arrange_scales, L.mi355moe_mxfp4_arranged_bytes
    assert size(2, 5, 96) == 80 and size(1, 3, 288) == 48
    for bad in ((0, 5, 96), (2, 0, 96), (2, 5, 40), (2, 5, 0), (2, 5, 1 << 17)):
        assert size(*bad) == -1 and f(P, *bad, P, NUL) == ESHAPE
    assert f(NUL, 1, 5, 96, P, NUL) == EINVAL and f(P, 1, 5, 96, NUL, NUL) == EINVAL and f(P, 1, 5, 96, ODD, NUL) == EINVAL


def test_gated_refusals(L):
    f = L.mi355moe_gated_forward

    def call(x=P, dt=BF16, T=4, H=64, xs=64, w=P, I=16, h=P, hs=16, gu=NUL, lim=10.0, ws=NUL, nb=0):
        return f(x, dt, T, H, xs, w, I, lim, h, hs, gu, ws, nb, NUL)

    assert call(dt=F32) == EDTYPE and call(lim=-1.0) == EINVAL and call(lim=float("nan")) == EINVAL
    assert call(H=60) == ESHAPE and call(I=12) == ESHAPE and call(T=-1) == ESHAPE and call(xs=56) == ESHAPE and call(hs=8) == ESHAPE
    assert call(T=1 << 25) == ELIMIT and call(H=1 << 17, xs=1 << 17) == ELIMIT
    assert call(x=NUL) == EINVAL and call(w=NUL) == EINVAL and call(h=NUL) == EINVAL
    assert call(h=ODD) == EINVAL and call(hs=20) == EINVAL
    assert call(x=ODD) == EINVAL and call(w=ODD) == EINVAL and call(xs=68) == EINVAL and call(gu=ODD) == EINVAL
    assert call(T=0, x=NUL) == 0
    need = L.mi355moe_gated_forward_workspace_bytes        # a cut contraction: fp32 sums of its parts
    cut = dict(T=120, H=4096, xs=4096, I=1024, hs=1024)
    nb = need(120, 4096, 1024)
    assert need(4, 64, 16) == 0 and need(4, 60, 16) == -1 and nb > 0 and need(8192, 4096, 1024) == 0
    assert call(**cut) == EINVAL and call(**cut, ws=ODD, nb=nb) == EINVAL and call(**cut, ws=P, nb=nb - 1) == EWORKSPACE
    b, size = L.mi355moe_gated_backward, L.mi355moe_gated_backward_workspace_bytes

    def back(dh=P, ds=16, gu=P, x=P, dt=BF16, T=4, H=64, xs=64, w=P, I=16, dx=P, dw=P, ws=P, nb=1 << 40):
        return b(dh, ds, gu, x, dt, T, H, xs, w, I, 10.0, dx, dw, ws, nb, NUL)

    assert back(dt=F32) == EDTYPE and back(ds=8) == ESHAPE and back(H=60) == ESHAPE
    assert back(T=0) == ESHAPE and back(T=0, dw=NUL) == 0 and back(dx=NUL, dw=NUL) == 0
    for k in ("dh", "gu", "x", "w", "ws"):
        assert back(**{k: NUL}) == EINVAL
    for k in ("dh", "gu", "x", "w", "dx", "dw", "ws"):
        assert back(**{k: ODD}) == EINVAL
    assert back(nb=size(4, 64, 16) - 1) == EWORKSPACE and size(4, 60, 16) == -1


def test_python_refusals():
    """Shape and type errors of the Python layer need no GPU: CPU tensors are refused first."""
    from mi355moe import ffn, mxfp4
    u8 = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        mxfp4.quant_rows(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="rows"):
        mxfp4.quant_rows(torch.zeros(32))
    with pytest.raises(ValueError, match="stride"):
        mxfp4.quant_rows(torch.zeros(32, 4).t())
    with pytest.raises(ValueError, match="overlap"):
        mxfp4.quant_rows(torch.zeros(1, 32).expand(4, 32))
    with pytest.raises(ValueError, match="GPU"):
        mxfp4.matmul(u8, u8[:, :2], u8, u8[:, :2])
    with pytest.raises(ValueError, match="uint8"):
        mxfp4.matmul(u8.int(), u8, u8, u8)
    w13, w2 = torch.zeros(2, 64, 32, dtype=torch.uint8), torch.zeros(2, 64, 16, dtype=torch.uint8)
    s13, s2 = torch.zeros(2, 64, 2, dtype=torch.uint8), torch.zeros(2, 64, 1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        mxfp4.Mxfp4Experts(w13, s13, w2, s2)
    with pytest.raises(ValueError, match="128"):
        mxfp4.Mxfp4Experts(w13, s13, w2, s2, arrange=False)
    big = [torch.zeros(s, dtype=torch.uint8) for s in ((2, 256, 128), (2, 256, 8), (2, 256, 64), (2, 256, 4))]
    ex = mxfp4.Mxfp4Experts(*big, arrange=False)
    assert (ex.n, ex.K, ex.N, ex.desc.arranged) == (2, 256, 128, 0)
    for bad in ((w13[:, :48], s13, w2, s2), (w13, s13[..., :1].contiguous(), w2, s2), (w13, s13, w2[:, :32].contiguous(), s2),
                (w13, s13, w2, s2.float()), (w13[..., ::2], s13, w2, s2), (w13[0], s13, w2, s2)):
        with pytest.raises(ValueError):
            mxfp4.Mxfp4Experts(*bad)
    with pytest.raises(ValueError, match="GPU"):
        mxfp4.moe_forward_ids(ex, torch.zeros(1, 256), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, 2))
    with pytest.raises(ValueError, match="GPU"):
        ffn.gated(torch.zeros(2, 64).half(), torch.zeros(32, 64).half())


def test_definitions():
    """The float64 definitions on values whose codes are known."""
    x = np.array([[0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] + [0.0] * 16], np.float32)
    q, s = ref.quant_rows(np.concatenate([x, -4 * x, x * 2.0 ** -130]))
    assert s[:, 0].tolist() == [127, 129, 0]
    v = ref.values(q, s, 32)
    assert v[0, :16].tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, 1, 1, 2, 2, 4, 4, 6]
    assert np.array_equal(v[1], -4 * v[0])
    assert np.array_equal(ref.rounded(x.astype(np.float64)), v[:1])
    assert v[2, 7] == 6 * 2.0 ** -130 * 1.0 or abs(v[2, 7] / (6 * 2.0 ** -130) - 1) <= 1 / 3
    h, _, _ = ref.swiglu(np.array([20.0]), np.array([-30.0]), 10.0)
    assert abs(h[0] + 100 / (1 + np.exp(-10.0))) < 1e-12
