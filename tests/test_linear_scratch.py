"""The workspace of the dense product's gradients is what the call uses: sizes, and the refusal of less. No GPU needed (refusals come
before any launch, and made-up addresses are never read)."""
from __future__ import annotations

import ctypes

import pytest

P, NUL = ctypes.c_void_p(0x10000), ctypes.c_void_p(0)
EINVAL, EWORKSPACE = 1, 4
F32, F16, BF16 = 0, 1, 2
NONE, RELU, SILU = 0, 1, 2


@pytest.fixture(scope="module")
def L():
    from mi355moe import _lib
    return _lib.lib()


def _up(n):
    return (n + 255) // 256 * 256


def test_sizes(L):
    size, full = L.mi355moe_linear_backward_call_bytes, L.mi355moe_linear_backward_workspace_bytes
    for K in (2560, 2563):                                       # outputs of so many tiles that no product is cut into parts
        M = N = 4096
        K8 = (K + 7) // 8 * 8
        dz, tops, db = _up(2 * M * N), _up(4 * 1025), _up(4 * (M // 64) * N)
        cx, cw = (0, 0) if K == K8 else (_up(2 * M * K8), _up(2 * N * K8))
        assert full(M, K, N) == dz + tops + cx + cw + db
        assert size(M, K, N, F16, SILU, 1, 1, 1, 1) == full(M, K, N)
        for act, aligned, takes in ((NONE, 1, 0), (NONE, 0, dz), (RELU, 1, dz), (SILU, 1, dz)):
            assert size(M, K, N, BF16, act, aligned, 1, 0, 0) == takes + cw
            assert size(M, K, N, BF16, act, aligned, 0, 1, 0) == takes + cx
            assert size(M, K, N, BF16, act, aligned, 1, 1, 1) == takes + cx + cw + db
            assert size(M, K, N, BF16, act, aligned, 0, 0, 1) == db and size(M, K, N, BF16, act, aligned, 0, 0, 0) == 0
            assert size(M, K, N, F16, act, aligned, 1, 0, 0) == takes + cw + (tops if act == SILU else 0)
    # dout of odd rows is copied whatever its address is
    assert size(4096, 2560, 4097, BF16, NONE, 1, 1, 0, 0) == _up(2 * 4096 * 4104)
    # parts are those of the products that are asked for: here of dW alone
    M, K, N = 8192, 1032, 1032
    assert size(M, K, N, BF16, NONE, 1, 1, 0, 0) == 0 < size(M, K, N, BF16, NONE, 1, 0, 1, 0) == size(M, K, N, BF16, NONE, 1, 1, 1, 0)
    # one size for a shape up to 1 MB
    for call in ((1, 1, 1, 1), (0, 1, 0, 0), (1, 0, 1, 1), (1, 0, 0, 0)):
        assert size(4, 64, 24, BF16, NONE, *call) == full(4, 64, 24)
    assert -1 == size(4, 64, 0, BF16, NONE, 1, 1, 1, 1) == size(4, 64, 24, F32, NONE, 1, 1, 1, 1) == size(4, 64, 24, BF16, 5, 1, 1, 1, 1)


def test_less_is_refused(L):
    M = N = 4096

    def back(nb, K=2560, ws=P, act=NONE, d=P, ds=N, dx=P, dw=P, db=P, dt=BF16):
        return L.mi355moe_linear_backward(d, ds, P, P, dt, M, K, 4096, P, N, 4096, act, dx, dw, db, F32, ws, nb, NUL)

    size = lambda *a, K=2560: L.mi355moe_linear_backward_call_bytes(M, K, N, *a)  # noqa: E731
    eight = ctypes.c_void_p(0x10008)
    for kw, need in ((dict(), size(BF16, NONE, 1, 1, 1, 1)), (dict(act=SILU, db=NUL), size(BF16, SILU, 1, 1, 1, 0)),
                     (dict(d=eight, db=NUL), size(BF16, NONE, 0, 1, 1, 0)), (dict(ds=N + 4, db=NUL), size(BF16, NONE, 0, 1, 1, 0)),
                     (dict(ds=1 << 23, db=NUL), size(BF16, NONE, 0, 1, 1, 0)), (dict(act=SILU, dt=F16, dw=NUL, db=NUL), size(F16, SILU, 1, 1, 0, 0)),
                     (dict(K=2563, dw=NUL, db=NUL), size(BF16, NONE, 1, 1, 0, 0, K=2563)), (dict(K=2563, dx=NUL), size(BF16, NONE, 1, 0, 1, 1, K=2563))):
        assert need > 0 and back(need - 1, **kw) == EWORKSPACE and back(0, **kw) == EWORKSPACE and back(need, ws=NUL, **kw) == EINVAL
