"""Refusals of the operators around a layer's experts: the C ABI's argument checks, which come before any launch (made-up
addresses are never read), what the Python layer refuses without a GPU, and the float64 definitions on known values."""
from __future__ import annotations

import ctypes
import types

import numpy as np
import pytest
import torch

from oracle import block as ref

P, NUL, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0), ctypes.c_void_p(0x10001)
TWO = ctypes.c_void_p(0x10002)
EINVAL, ESHAPE, ELIMIT, EWORKSPACE, EDTYPE = 1, 2, 3, 4, 5
F32, F16, BF16, I32, I64 = range(5)


@pytest.fixture(scope="module")
def L():
    from mi355moe import _lib
    return _lib.lib()


def test_sort_refusals(L):
    size = L.mi355moe_sort_tokens_workspace_bytes

    def call(ids=P, dt=I32, T=4, k=2, em=NUL, ng=0, n=8, row=P, pair=P, off=P, ws=P, nb=1 << 30):
        return L.mi355moe_sort_tokens(ids, dt, T, k, em, ng, n, row, pair, off, ws, nb, NUL)

    assert call(dt=F32) == EDTYPE and call(T=-1) == ESHAPE
    assert call(k=0) == ELIMIT and call(k=33) == ELIMIT and call(T=1 << 24, k=2) == ELIMIT and call(T=(1 << 24) + 1, k=1) == ELIMIT
    assert call(n=0) == ELIMIT and call(n=4097) == ELIMIT and call(em=P, ng=-1) == EINVAL
    for k in ("ids", "row", "pair", "off"):
        assert call(**{k: NUL}) == EINVAL
    assert size(4, 2, 8) == 0 and size(4096, 1, 8) == 0 and size(-1, 2, 8) == -1 and size(4, 0, 8) == -1 and size(4, 2, 0) == -1
    nb = size(1000, 8, 288)
    assert nb == 4 * 8 * 289 and size(1 << 21, 8, 288) == 4 * 128 * 289 and size(1 << 21, 8, 4096) == 4 * 32 * 4097
    big = dict(T=1000, k=8, n=288)
    assert call(**big, ws=NUL) == EINVAL and call(**big, ws=ODD) == EINVAL and call(**big, nb=nb - 1) == EWORKSPACE


def test_rows_refusals(L):
    def to(x=P, dt=BF16, T=4, H=16, xs=16, row=P, k=2, rows=P):
        return L.mi355moe_rows_to_experts(x, dt, T, H, xs, row, k, rows, NUL)

    def back(rows=P, dt=BF16, T=4, H=16, row=P, k=2, w=P, wdt=F32, sh=NUL, ss=0, out=P, os=16):
        return L.mi355moe_rows_from_experts(rows, dt, T, H, row, k, w, wdt, sh, ss, out, os, NUL)

    def grad(d=P, dt=BF16, T=4, H=16, ds=16, row=P, k=2, w=P, wdt=F32, rows=P, dr=P, dw=P):
        return L.mi355moe_rows_from_experts_backward(d, dt, T, H, ds, row, k, w, wdt, rows, dr, dw, NUL)

    for f in (to, back, grad):
        assert f(dt=I32) == EDTYPE and f(T=-1) == ESHAPE and f(H=0) == ESHAPE and f(k=0) == ELIMIT and f(k=33) == ELIMIT
        assert f(T=1 << 23, k=3) == ELIMIT
    assert to(H=65537, xs=65537) == ELIMIT and to(xs=15) == ESHAPE and back(os=15) == ESHAPE and back(sh=P, ss=15) == ESHAPE and grad(ds=15) == ESHAPE
    for k in ("x", "row", "rows"):
        assert to(**{k: NUL}) == EINVAL
    for k in ("rows", "row", "out"):
        assert back(**{k: NUL}) == EINVAL
    for k in ("d", "row", "w", "rows"):
        assert grad(**{k: NUL}) == EINVAL
    assert back(wdt=I32) == EDTYPE and grad(wdt=I64) == EDTYPE and back(w=NUL, wdt=I32, T=0) == 0
    assert to(T=0, x=NUL) == 0 and back(T=0, out=NUL) == 0 and grad(T=0) == 0 and grad(dr=NUL, dw=NUL) == 0
    # an address that is none of the type's
    assert to(x=ODD) == EINVAL and to(rows=ODD) == EINVAL and back(out=ODD) == EINVAL and back(sh=ODD, ss=16) == EINVAL
    assert grad(d=ODD) == EINVAL and grad(dr=ODD) == EINVAL and to(dt=F32, x=TWO) == EINVAL and back(rows=TWO, dt=F32) == EINVAL


def test_linear_refusals(L):
    size, bsize = L.mi355moe_linear_forward_workspace_bytes, L.mi355moe_linear_backward_workspace_bytes

    def call(x=P, dt=BF16, M=4, K=64, xs=64, w=P, N=24, wst=64, b=NUL, bdt=F32, act=0, r=NUL, rs=0, out=P, os=24, z=NUL, ws=P, nb=1 << 40):
        return L.mi355moe_linear_forward(x, dt, M, K, xs, w, N, wst, b, bdt, act, r, rs, out, os, z, ws, nb, NUL)

    def back(d=P, ds=24, z=P, x=P, dt=BF16, M=4, K=64, xs=64, w=P, N=24, wst=64, act=0, dx=P, dw=P, db=P, bdt=F32, ws=P, nb=1 << 40):
        return L.mi355moe_linear_backward(d, ds, z, x, dt, M, K, xs, w, N, wst, act, dx, dw, db, bdt, ws, nb, NUL)

    for f in (call, back):
        assert f(dt=F32) == EDTYPE and f(M=-1) == ESHAPE and f(K=0, xs=64, wst=64) == ESHAPE and f(N=0) == ESHAPE
        assert f(M=(1 << 24) + 1) == ELIMIT and f(K=65544, xs=65544, wst=65544) == ELIMIT and f(act=5) == EINVAL and f(act=-1) == EINVAL
        assert f(xs=56) == ESHAPE and f(wst=56) == ESHAPE and f(xs=(1 << 22) + 8) == ESHAPE and f(wst=(1 << 22) + 8) == ESHAPE
        assert f(x=NUL) == EINVAL and f(w=NUL) == EINVAL
        assert f(x=TWO) == EINVAL and f(w=TWO) == EINVAL and f(xs=68) == EINVAL and f(wst=68) == EINVAL      # K % 8 == 0: whole 16 bytes
        assert f(K=63, xs=64, wst=64, x=ODD) == EINVAL
    assert call(N=(1 << 18) + 1, os=1 << 19) == ELIMIT and call(os=23) == ESHAPE and call(r=P, rs=23) == ESHAPE and call(b=P, bdt=I32) == EDTYPE
    assert call(out=NUL) == EINVAL and call(out=ODD) == EINVAL and call(r=ODD, rs=24) == EINVAL and call(z=TWO) == EINVAL and call(b=TWO) == EINVAL
    assert call(M=0, x=NUL, out=NUL) == 0
    assert size(4, 64, 24) == 0 and size(4, 0, 24) == -1 and size(4, 64, 0) == -1
    cut = dict(M=130, K=4104, xs=4104, wst=4104, N=1032, os=1032)
    nb = size(130, 4104, 1032)
    assert nb > 0 and call(**cut, ws=NUL) == EINVAL and call(**cut, ws=ODD) == EINVAL and call(**cut, nb=nb - 1) == EWORKSPACE
    odd = size(4100, 1027, 2051)
    assert size(900, 131, 777) == 0 and odd == (4100 * 1032 * 2 + 255) // 256 * 256 + (2051 * 1032 * 2 + 255) // 256 * 256
    assert back(ds=23) == ESHAPE and back(db=P, bdt=I32) == EDTYPE and back(d=NUL) == EINVAL and back(ws=NUL) == EINVAL and back(ws=ODD) == EINVAL
    assert back(act=2, z=NUL) == EINVAL and back(d=ODD) == EINVAL and back(dx=ODD) == EINVAL and back(dw=ODD) == EINVAL and back(db=TWO) == EINVAL
    assert back(act=2, z=TWO) == EINVAL
    assert back(dx=NUL, dw=NUL, db=NUL) == 0 and back(M=0) == ESHAPE and back(M=0, dw=NUL, db=NUL) == 0
    assert back(nb=bsize(4, 64, 24) - 1) == EWORKSPACE and bsize(4, 64, 0) == -1


def test_norm_refusals(L):
    size = L.mi355moe_norm_backward_workspace_bytes

    def call(b=P, dt=BF16, R=4, H=64, bs=64, r=NUL, rs=0, post=NUL, pre=P, wdt=F32, g=NUL, gdt=F32, kind=0, eps=1e-5, s=P, y=P, st=NUL):
        return L.mi355moe_norm_forward(b, dt, R, H, bs, r, rs, post, pre, wdt, g, gdt, kind, eps, 1.0, 1.0, s, y, st, NUL)

    def back(ds=P, dss=64, dy=P, dys=64, b=P, dt=BF16, R=4, H=64, bs=64, r=NUL, rs=0, post=P, pre=P, wdt=F32, g=P, gdt=F32, kind=1, st=P,
             db=P, dr=P, dpo=P, dpr=P, dg=P, ws=P, nb=1 << 40):
        return L.mi355moe_norm_backward(ds, dss, dy, dys, b, dt, R, H, bs, r, rs, post, pre, wdt, g, gdt, kind, 1.0, 1.0, st, db, dr, dpo, dpr,
                                        dg, ws, nb, NUL)

    for f in (call, back):
        assert f(dt=I32) == EDTYPE and f(R=-1) == ESHAPE and f(H=0, bs=64) == ESHAPE and f(H=16385, bs=16385) == ELIMIT
        assert f(R=(1 << 26) + 1) == ELIMIT and f(wdt=I32) == EDTYPE and f(bs=63) == ESHAPE and f(r=P, rs=63) == ESHAPE
        assert f(g=P, kind=0) == EINVAL and f(g=NUL, kind=1) == EINVAL and f(g=P, kind=4) == EINVAL and f(g=P, kind=-1) == EINVAL
        assert f(g=P, kind=2, gdt=I32) == EDTYPE and f(b=NUL) == EINVAL and f(b=ODD) == EINVAL and f(g=ODD, kind=1) == EINVAL
        assert f(pre=TWO) == EINVAL and f(post=TWO) == EINVAL and f(r=ODD, rs=64) == EINVAL
    assert call(eps=-1.0) == EINVAL and call(eps=float("nan")) == EINVAL and call(pre=NUL) == EINVAL and call(y=NUL) == EINVAL
    assert call(pre=NUL, y=NUL, s=NUL) == EINVAL and call(s=ODD) == EINVAL and call(y=ODD) == EINVAL and call(st=TWO) == EINVAL
    assert call(R=0, b=NUL) == 0
    assert back(dss=63) == ESHAPE and back(dys=63) == ESHAPE and back(pre=NUL) == EINVAL and back(dy=NUL) == EINVAL and back(post=NUL) == EINVAL
    assert back(ds=NUL, dy=NUL, dpr=NUL) == EINVAL and back(st=NUL) == EINVAL and back(g=NUL, kind=0) == EINVAL
    for k in ("ds", "dy", "db", "dr", "dg"):
        assert back(**{k: ODD}) == EINVAL
    for k in ("dpo", "dpr", "st"):
        assert back(**{k: TWO}) == EINVAL
    none = dict(db=NUL, dr=NUL, dpo=NUL, dpr=NUL, dg=NUL)
    assert back(**none) == 0 and back(R=0) == ESHAPE and back(R=0, dpo=NUL, dpr=NUL, dg=NUL) == 0
    assert back(ws=NUL) == EINVAL and back(ws=ODD) == EINVAL and back(nb=size(4, 64) - 1) == EWORKSPACE
    assert size(4, 64) == 4 * 2 * 64 and size(33, 64) == 2 * 4 * 2 * 64 and size(4, 600) == 4 * 4 * 2 * 600 and size(1 << 20, 4096) == 4 * 512 * 2 * 4096 and size(4, 0) == -1


def test_python_refusals():
    """CPU tensors are refused; what the calls say of shapes and types needs a GPU (tests/test_gpu_block_args.py)."""
    from mi355moe import dispatch, ffn, norm
    x = torch.zeros(2, 8).half()
    with pytest.raises(ValueError, match="GPU"):
        dispatch.sort_tokens(torch.zeros(2, 2, dtype=torch.int32), 4)
    plan = dispatch.SortedTokens(torch.zeros(16, dtype=torch.int32), 2, 2, 4)
    for f in (lambda: dispatch.to_experts(x, plan), lambda: dispatch.from_experts(torch.zeros(4, 8), None, plan),
              lambda: dispatch.from_experts_backward(torch.zeros(2, 8), torch.zeros(4, 8), torch.zeros(2, 2), plan),
              lambda: ffn.linear(x, x), lambda: ffn.linear_forward(x, x), lambda: ffn.linear_backward(x, None, x, x),
              lambda: norm.join(x), lambda: norm.join_forward(x), lambda: norm.rms(x, x[0]),
              lambda: norm.join_backward(x, None, torch.zeros(2, 2), x)):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_backward_is_refused_during_capture(monkeypatch):
    """The backward pass of an eager call while a graph is captured: refused before anything is launched (the capture is pretended:
    what such a one would record is not a thing to try on a GPU)."""
    from mi355moe import dispatch, ffn, norm

    def launched(*a, **k):
        raise AssertionError("launched")

    t = torch.zeros(2, 16)
    six = types.SimpleNamespace(saved_tensors=(t,) * 6, rest=((t.device, 0, 0, 0, 0), 1.0, 1.0, True, True), needs_input_grad=(True,) * 10)
    three = types.SimpleNamespace(saved_tensors=(t,) * 3, rest=((t.device, 0, 0), None, None), needs_input_grad=(True, True, False, False, False, False))
    two = types.SimpleNamespace(saved_tensors=(t, t), rest=(t.device, 0, None), needs_input_grad=(True, True, False, False))
    for mod, fn, inner, ctx, grads in ((norm, norm._Join, "_backward", six, (t, t)), (ffn, ffn._Linear, "_linear_grads", three, (t,)),
                                       (dispatch, dispatch._From, "_from_grads", two, (t,)), (dispatch, dispatch._To, "_gather", two, (t,))):
        monkeypatch.setattr(mod, inner, launched)
        monkeypatch.setattr(mod, "_capturing", lambda dev: True)
        for enabled in (False, True):
            with torch.set_grad_enabled(enabled), pytest.raises(RuntimeError, match="capture"):
                fn.backward(ctx, *grads)
        monkeypatch.setattr(mod, "_capturing", lambda dev: False)
        with torch.no_grad(), pytest.raises(AssertionError, match="launched"):
            fn.backward(ctx, *grads)


def test_views_of_rows():
    """What goes to the kernels of a user's views: the address and stride that the C layer takes, a copy only where it must be."""
    from mi355moe import ffn, ops
    base = torch.zeros(40, 64, dtype=torch.float16)
    for t, kept, ld in ((base, True, 64), (base[:, 3:50], True, 64), (base[5:6, 3:50], True, 47), (base[::2], True, 128), (base.t(), False, 40),
                        (base[:1].expand(4, 64), False, 64), (base[:, :1], True, 64), (base.view(4, 10, 64), True, 64),
                        (base[:, ::2], False, 32), (base.view(4, 10, 64)[:, 0], True, 640), (base.view(4, 10, 64)[:, :5], False, 64), (base[0], True, 64)):
        r, stride = ops._rows_any(t)
        assert (r.data_ptr() == t.data_ptr()) == kept and stride == ld and r.reshape(t.shape).equal(t)
        assert r.numel() == 0 or r.shape[-1] == t.shape[-1]
    leaf = base.clone().requires_grad_()
    assert ops._rows_any(leaf)[0] is leaf and not ops._rows_any(leaf.t())[0].requires_grad and ops._packed(leaf) is leaf
    one = torch.empty_strided((1, 64), (8388608, 1), dtype=torch.float16)
    assert ops._rows_any(one)[1] == 64 and ffn._linear_operand(one, 64)[1] == 64
    far = torch.empty(0, dtype=torch.float16)
    assert ops._rows_any(far.view(0, 7)) [1] == 7
    for t in (base[:, 3:11], base[:, :64][:, 1:9], base[1:, :8]):
        r, ld = ffn._linear_operand(t, 8)
        assert r.data_ptr() % 16 == 0 and ld % 8 == 0 and torch.equal(r, t)
    r, ld = ffn._linear_operand(base[:, 3:12], 9)
    assert r.data_ptr() == base[:, 3:12].data_ptr() and ld == 64


def test_definitions():
    row, pair, offsets = ref.order([[2, 0], [5, 2], [-1, 0]], 3)
    assert row.tolist() == [[2, 0], [~4, 3], [~5, 1]] and pair.tolist() == [1, 5, 0, 3, ~2, ~4] and offsets.tolist() == [0, 2, 2, 4]
    row, _, _ = ref.order([[2, 0]], 3, [1, 0, -1])
    assert row.tolist() == [[~1, 0]]
    for name in ("silu", "gelu", "gelu_tanh"):
        z = np.linspace(-6, 6, 49)
        y, slope, _ = ref.act(name, z)
        step = 1e-6
        assert np.abs((ref.act(name, z + step)[0] - ref.act(name, z - step)[0]) / (2 * step) - slope).max() < 1e-8
        assert np.abs(y - getattr(torch.nn.functional, name.split("_")[0])(torch.tensor(z), **({"approximate": "tanh"} if "_" in name else {})).numpy()).max() < 1e-12
    x = np.array([[3.0, 4.0]])
    (s, _), (y, _) = ref.norm(x, None, None, None, np.ones(2), 0.0, 1.0, 1.0, 0.0, 0.0)
    assert np.allclose(s, x) and np.allclose(y, x / np.sqrt(12.5))
