"""What the GroupNorm, quantiser and 8-bit product entries refuse, and their empty calls: all decided on the host, before any device
work."""
import ctypes

import pytest

from sdvk_amd import _lib

FAKE = 1 << 20
GAP = 1 << 36  # between made-up tensors: larger than any of them
INVALID, UNSUPPORTED, ALIGN, ALIAS = _lib.MI_ERR_INVALID_ARG, _lib.MI_ERR_UNSUPPORTED, _lib.MI_ERR_ALIGNMENT, _lib.MI_ERR_ALIASING


def addr(i):
    return FAKE + i * GAP


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def norm_args(**kw):
    a = dict(x=addr(0), gamma=addr(1), beta=addr(2), y=addr(3), y_scale=None, stats=addr(4), batch=2, pixels=50, channels=64, groups=8,
             x_dtype=0, y_dtype=0, act=1, eps=1e-5)
    a.update(kw)
    return _lib.MiGroupnormArgs(**a)


def norm(lib, ws=addr(9), ws_bytes=1 << 20, **kw):
    return lib.mi_groupnorm(ctypes.byref(norm_args(**kw)), ws, ws_bytes, None)


def test_groupnorm(lib):
    assert lib.mi_groupnorm(None, None, 0, None) == INVALID
    assert norm(lib, batch=0, ws=None) == _lib.MI_OK and norm(lib, pixels=0, x=None, ws=None) == _lib.MI_OK
    nan, inf = float("nan"), float("inf")
    for bad in (dict(x=None), dict(y=None), dict(x_dtype=2), dict(y_dtype=3), dict(y_dtype=2), dict(y_scale=addr(5)), dict(act=2), dict(eps=nan), dict(eps=-1e-5),
                dict(eps=inf), dict(channels=0), dict(groups=0), dict(groups=7), dict(ldx=63), dict(ldy=63), dict(ws=None), dict(ws_bytes=64),
                dict(ldy=64, sy=50 * 64 - 1), dict(ldy=127, sy=64), dict(ldy=128, sy=63), dict(pixels=1, sy=63)):
        assert norm(lib, **bad) == INVALID, bad
    for bad in (dict(batch=(1 << 20) + 1, pixels=1), dict(batch=2, pixels=(1 << 30) + 1), dict(channels=1 << 21, groups=1), dict(ldx=1 << 60), dict(sx=1 << 61),
                dict(ldy=1 << 60, sy=64)):
        assert norm(lib, **bad) == UNSUPPORTED, bad
    for bad in (dict(x=addr(0) + 2), dict(x=addr(0) + 1, x_dtype=1), dict(y=addr(3) + 2), dict(y=addr(3) + 1, y_dtype=1), dict(gamma=addr(1) + 2), dict(beta=addr(2) + 1),
                dict(stats=addr(4) + 4), dict(ws=addr(9) + 8), dict(y_dtype=2, y_scale=addr(5) + 2)):
        assert norm(lib, **bad) == ALIGN, bad
    for bad in (dict(y=addr(0)), dict(y=addr(0) + 2 * 50 * 64 * 4 - 4), dict(y=addr(1)), dict(y=addr(2)), dict(stats=addr(0) + 16), dict(stats=addr(3)), dict(ws=addr(0)),
                dict(ws=addr(3) + 16), dict(ws=addr(4)), dict(y_dtype=2, y_scale=addr(3)), dict(y_dtype=2, y_scale=addr(0)), dict(ws=addr(1))):
        assert norm(lib, **bad) == ALIAS, bad
    assert lib.mi_groupnorm_ws_bytes(2, 50, 64, 7) == 0 and lib.mi_groupnorm_ws_bytes(2, 50, 0, 1) == 0 and lib.mi_groupnorm_ws_bytes(2, 0, 64, 8) == 0
    assert lib.mi_groupnorm_ws_bytes((1 << 20) + 1, 1, 64, 8) == 0
    need = lib.mi_groupnorm_ws_bytes(2, 50, 64, 8)
    assert need > 0 and norm(lib, ws_bytes=need - 1) == INVALID
    assert ctypes.sizeof(_lib.MiGroupnormArgs) == 6 * 8 + 8 * 4 + 4 * 8


def bwd(lib, ws=addr(9), ws_bytes=1 << 20, **kw):
    g = dict(dy=addr(5), res=addr(6), dx=addr(7), dgamma=addr(8), dbeta=addr(10))
    f = dict(y=None)
    for name, v in kw.items():
        (g if name in dict(_lib.MiGroupnormBwdArgs._fields_) else f)[name] = v
    x = _lib.MiGroupnormBwdArgs(fwd=norm_args(**f), **g)
    return lib.mi_groupnorm_bwd(ctypes.byref(x), ws, ws_bytes, None)


def test_groupnorm_bwd(lib):
    assert lib.mi_groupnorm_bwd(None, None, 0, None) == INVALID
    assert bwd(lib, pixels=0, dgamma=None, dbeta=None, ws=None) == _lib.MI_OK
    for bad in (dict(x=None), dict(dy=None), dict(dx=None), dict(y_dtype=2), dict(x_dtype=3), dict(act=-1), dict(dgamma=None), dict(dbeta=None), dict(lddy=63), dict(ldres=63),
                dict(lddx=63), dict(ldx=1), dict(ws=None), dict(ws_bytes=100), dict(groups=3), dict(lddx=64, sdx=100)):
        assert bwd(lib, **bad) == INVALID, bad
    for bad in (dict(batch=1 << 21), dict(lddy=1 << 60), dict(sres=1 << 61), dict(sdx=1 << 61)):
        assert bwd(lib, **bad) == UNSUPPORTED, bad
    for bad in (dict(x=addr(0) + 2), dict(dy=addr(5) + 1, y_dtype=1), dict(dx=addr(7) + 2), dict(res=addr(6) + 1), dict(dgamma=addr(8) + 2), dict(dbeta=addr(10) + 1), dict(ws=addr(9) + 8),
                dict(stats=addr(4) + 8)):
        assert bwd(lib, **bad) == ALIGN, bad
    for bad in (dict(dx=addr(0)), dict(dx=addr(5)), dict(dx=addr(6) + 16), dict(dx=addr(1)), dict(dx=addr(4)), dict(dgamma=addr(7)), dict(dbeta=addr(8)), dict(dgamma=addr(1)), dict(ws=addr(0)),
                dict(ws=addr(7)), dict(ws=addr(10)), dict(ws=addr(4)), dict(dx=addr(6), lddx=72)):
        assert bwd(lib, **bad) == ALIAS, bad
    assert lib.mi_groupnorm_bwd_ws_bytes(2, 50, 64, 7) == 0 and lib.mi_groupnorm_bwd_ws_bytes(2, 50, 64, 8) > lib.mi_groupnorm_ws_bytes(2, 50, 64, 8)
    assert ctypes.sizeof(_lib.MiGroupnormBwdArgs) == ctypes.sizeof(_lib.MiGroupnormArgs) + 5 * 8 + 6 * 8


def test_quantize(lib):
    def call(x=addr(0), dtype=0, q=addr(1), scale=addr(2), rows=5, cols=64, ldx=0, ldq=0):
        return lib.mi_quantize_rows_i8(x, dtype, q, scale, rows, cols, ldx, ldq, None)

    assert call(rows=0, x=None) == _lib.MI_OK and call(cols=0, q=None) == _lib.MI_OK
    for bad in (dict(x=None), dict(q=None), dict(scale=None), dict(dtype=2), dict(dtype=-1), dict(ldx=63), dict(ldq=63)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(rows=(1 << 31) + 1, cols=1), dict(rows=1, cols=(1 << 30) + 1)):
        assert call(**bad) == UNSUPPORTED, bad
    for bad in (dict(x=addr(0) + 2), dict(x=addr(0) + 1, dtype=1), dict(scale=addr(2) + 2)):
        assert call(**bad) == ALIGN, bad
    for bad in (dict(q=addr(0)), dict(q=addr(0) + 5 * 64 * 4 - 1), dict(scale=addr(0) + 4), dict(scale=addr(1) + 4)):
        assert call(**bad) == ALIAS, bad


def test_product(lib):
    def call(A=addr(0), sa=addr(1), W=addr(2), sw=addr(3), bias=addr(4), C=addr(5), dt=0, M=8, N=8, K=64, mode=0, lda=0, ldw=0, ldc=0):
        return lib.mi_gemm_nt_i8(A, sa, W, sw, bias, C, dt, M, N, K, mode, lda, ldw, ldc, None)

    assert call(M=0, A=None) == _lib.MI_OK and call(N=0, K=0) == _lib.MI_OK
    for bad in (dict(A=None), dict(sa=None), dict(W=None), dict(sw=None), dict(C=None), dict(dt=2), dict(mode=3), dict(lda=63), dict(ldw=63), dict(ldc=7)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(K=0), dict(K=131072), dict(M=(1 << 31) + 1), dict(N=(1 << 31) + 1)):
        assert call(**bad) == UNSUPPORTED, bad
    for bad in (dict(sa=addr(1) + 2), dict(sw=addr(3) + 1), dict(bias=addr(4) + 2), dict(C=addr(5) + 2), dict(C=addr(5) + 1, dt=1)):
        assert call(**bad) == ALIGN, bad
    for bad in (dict(C=addr(0)), dict(C=addr(1)), dict(C=addr(2) + 64), dict(C=addr(3)), dict(C=addr(4) + 28)):
        assert call(**bad) == ALIAS, bad


def test_plan_override(lib):
    assert lib.mi_tuning_set(b"gemm_i8_cfg", b"8") == _lib.MI_OK
    for bad in (b"9", b"-1", b"x", b"1:2"):
        assert lib.mi_tuning_set(b"gemm_i8_cfg", bad) == INVALID, bad
    assert lib.mi_tuning_set(b"gemm_i8_cfg", None) == _lib.MI_OK
    lib.mi_tuning_reset()
