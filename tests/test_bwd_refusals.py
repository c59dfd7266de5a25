"""What the backward entries refuse, and their empty calls: all decided on the host, before any device work."""
import pytest

from sdvk_amd import _lib

FAKE = 1 << 20
GAP = 1 << 32  # between made-up tensors: larger than any of them


def addr(i):
    return FAKE + i * GAP


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def linear(lib, dC=addr(0), W=addr(1), dA=addr(2), dtype=1, M=64, N=64, K=64, mode=0, ldc=0, lda=0, ws=None, ws_bytes=0):
    return lib.mi_gemm_nt_q8_0_bwd(dC, W, dA, dtype, M, N, K, mode, ldc, lda, ws, ws_bytes, None)


def test_linear(lib):
    assert linear(lib, M=0) == _lib.MI_OK and linear(lib, K=0) == _lib.MI_OK
    assert linear(lib, N=0, mode=1, dC=None, W=None) == _lib.MI_OK
    for bad in (dict(dC=None), dict(W=None), dict(dA=None), dict(dtype=2), dict(mode=2), dict(ldc=63), dict(lda=63)):
        assert linear(lib, **bad) == _lib.MI_ERR_INVALID_ARG, bad
    assert linear(lib, K=48) == _lib.MI_ERR_UNSUPPORTED
    assert linear(lib, N=1 << 20, K=2048) == _lib.MI_ERR_UNSUPPORTED          # a weight of 2 GiB
    assert linear(lib, ldc=1 << 23) == _lib.MI_ERR_UNSUPPORTED                # 256 rows past 2 GiB
    assert linear(lib, M=1 << 31, K=1 << 12) == _lib.MI_ERR_UNSUPPORTED
    for bad in (dict(W=addr(1) + 8), dict(dC=addr(0) + 1), dict(dA=addr(2) + 1), dict(dA=addr(2) + 2, dtype=0)):
        assert linear(lib, **bad) == _lib.MI_ERR_ALIGNMENT, bad
    assert linear(lib, dA=addr(0)) == _lib.MI_ERR_ALIASING and linear(lib, dA=addr(1) + 32) == _lib.MI_ERR_ALIASING
    need = lib.mi_gemm_nt_q8_0_bwd_ws_bytes(64, 1280, 64, 1)
    assert need > 0 and lib.mi_gemm_nt_q8_0_bwd_ws_bytes(64, 1280, 48, 1) == 0 and lib.mi_gemm_nt_q8_0_bwd_ws_bytes(64, 1280, 64, 7) == 0
    assert linear(lib, N=1280, ws=addr(3) + 4, ws_bytes=need) == _lib.MI_ERR_ALIGNMENT
    for at in (0, 1, 2):
        assert linear(lib, N=1280, ws=addr(at), ws_bytes=need) == _lib.MI_ERR_ALIASING


def test_geglu(lib):
    def call(h=addr(0), dy=addr(1), dh=addr(2), dtype=0, rows=4, F=64):
        return lib.mi_geglu_bwd(h, dy, dh, dtype, rows, F, None)

    assert call(rows=0) == _lib.MI_OK and call(F=0) == _lib.MI_OK
    for bad in (dict(h=None), dict(dy=None), dict(dh=None), dict(dtype=3)):
        assert call(**bad) == _lib.MI_ERR_INVALID_ARG, bad
    assert call(rows=(1 << 31) + 1, F=1) == _lib.MI_ERR_UNSUPPORTED
    for bad in (dict(h=addr(0) + 2), dict(dy=addr(1) + 2), dict(dh=addr(2) + 1, dtype=1)):
        assert call(**bad) == _lib.MI_ERR_ALIGNMENT, bad
    for bad in (dict(dh=addr(1)), dict(dh=addr(0) + 16), dict(dh=addr(0), dtype=1)):
        assert call(**bad) == _lib.MI_ERR_ALIASING, bad


def test_geglu_gemm(lib):
    def call(A=addr(0), W=addr(1), bias=addr(2), dG=addr(3), dH=addr(4), M=64, F=64, K=64, lda=0, lddg=0, lddh=0):
        return lib.mi_gemm_nt_q8_0_geglu_bwd(A, W, bias, dG, dH, M, F, K, lda, lddg, lddh, None)

    assert call(M=0) == _lib.MI_OK and call(F=0) == _lib.MI_OK
    for bad in (dict(A=None), dict(W=None), dict(dG=None), dict(dH=None), dict(lda=56), dict(lddg=63), dict(lddh=127)):
        assert call(**bad) == _lib.MI_ERR_INVALID_ARG, bad
    for bad in (dict(K=0), dict(K=48), dict(F=(1 << 30) + 1), dict(F=1 << 20, K=2048)):
        assert call(**bad) == _lib.MI_ERR_UNSUPPORTED, bad
    for bad in (dict(A=addr(0) + 8), dict(lda=68), dict(W=addr(1) + 4), dict(dG=addr(3) + 1), dict(dH=addr(4) + 2)):
        assert call(**bad) == _lib.MI_ERR_ALIGNMENT, bad
    for i in range(4):
        assert call(dH=addr(i)) == _lib.MI_ERR_ALIASING, i


def test_layernorm(lib):
    def call(x=addr(0), gamma=addr(1), dy=addr(2), dt=0, res=addr(3), dx=addr(4), dg=addr(5), db=addr(6), rows=8, d=64, ws=addr(7),
             ws_bytes=1 << 20):
        return lib.mi_layernorm_bwd(x, gamma, dy, dt, res, dx, dg, db, rows, d, 1e-5, ws, ws_bytes, None)

    assert call(rows=0, dg=None, db=None) in (_lib.MI_OK, _lib.MI_ERR_HIP)  # nothing to launch (no device here)
    for bad in (dict(x=None), dict(dy=None), dict(dx=None), dict(dt=5), dict(dg=None), dict(db=None), dict(d=0), dict(ws=None), dict(ws_bytes=64)):
        assert call(**bad) == _lib.MI_ERR_INVALID_ARG, bad
    assert call(rows=(1 << 31) + 1, d=1) == _lib.MI_ERR_UNSUPPORTED
    for bad in (dict(x=addr(0) + 2), dict(gamma=addr(1) + 2), dict(dy=addr(2) + 1, dt=1), dict(dx=addr(4) + 2), dict(res=addr(3) + 1),
                dict(dg=addr(5) + 2), dict(ws=addr(7) + 8)):
        assert call(**bad) == _lib.MI_ERR_ALIGNMENT, bad
    for bad in (dict(dx=addr(0)), dict(dx=addr(2)), dict(dx=addr(3) + 16), dict(dx=addr(1)), dict(dg=addr(4)), dict(db=addr(5)), dict(dg=addr(1)),
                dict(ws=addr(0)), dict(ws=addr(4)), dict(ws=addr(6))):
        assert call(**bad) == _lib.MI_ERR_ALIASING, bad
