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
    assert call(rows=1, d=(1 << 30) + 1) == _lib.MI_ERR_UNSUPPORTED  # the columns are counted in 32 bits
    for bad in (dict(x=addr(0) + 2), dict(gamma=addr(1) + 2), dict(dy=addr(2) + 1, dt=1), dict(dx=addr(4) + 2), dict(res=addr(3) + 1),
                dict(dg=addr(5) + 2), dict(ws=addr(7) + 8)):
        assert call(**bad) == _lib.MI_ERR_ALIGNMENT, bad
    for bad in (dict(dx=addr(0)), dict(dx=addr(2)), dict(dx=addr(3) + 16), dict(dx=addr(1)), dict(dg=addr(4)), dict(db=addr(5)), dict(dg=addr(1)),
                dict(ws=addr(0)), dict(ws=addr(4)), dict(ws=addr(6))):
        assert call(**bad) == _lib.MI_ERR_ALIASING, bad


def attn(lib, ws=addr(20), ws_bytes=None, **kw):
    import ctypes

    a = dict(q=addr(0), k=addr(1), v=addr(2), out=addr(3), batch=2, Tq=64, Tk=64, C=128, heads=2, in_dtype=1, out_dtype=1)
    g = dict(dout=addr(4), dq=addr(5), dk=addr(6), dv=addr(7))
    for name, v in kw.items():
        (g if name in dict(_lib.MiAttnBwdArgs._fields_) else a)[name] = v
    x = _lib.MiAttnBwdArgs(fwd=_lib.MiAttnArgs(**a), **g)
    need = lib.mi_fused_attention_bwd_ws_bytes(ctypes.byref(x))
    return lib.mi_fused_attention_bwd(ctypes.byref(x), ws, need if ws_bytes is None else ws_bytes, None)


def test_attention(lib):
    import ctypes

    assert lib.mi_fused_attention_bwd(None, None, 0, None) == _lib.MI_ERR_INVALID_ARG
    assert lib.mi_fused_attention_bwd_ws_bytes(None) == 0
    assert attn(lib, Tq=0, Tk=0, ws=None) == _lib.MI_OK
    for bad in (dict(in_dtype=2), dict(out_dtype=0), dict(batch=0), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(dout=None),
                dict(dq=None), dict(dk=None), dict(dv=None), dict(scale=float("inf")), dict(scale=float("nan")), dict(ldq=100), dict(lddk=64),
                dict(sdq=100), dict(sdv=8000), dict(ws=None), dict(ws_bytes=100)):
        assert attn(lib, **bad) == _lib.MI_ERR_INVALID_ARG, bad
    for bad in (dict(C=130), dict(heads=3), dict(C=129, heads=1), dict(batch=70000), dict(ldk=1 << 22), dict(lddq=1 << 22),
                dict(Tq=1 << 26, C=2, batch=8)):
        assert attn(lib, **bad) == _lib.MI_ERR_UNSUPPORTED, bad
    for bad in (dict(q=addr(0) + 1), dict(dv=addr(7) + 1), dict(ws=addr(20) + 8)):
        assert attn(lib, **bad) == _lib.MI_ERR_ALIGNMENT, bad
    for bad in (dict(dq=addr(0)), dict(dk=addr(3)), dict(dv=addr(4) + 64), dict(dk=addr(5)), dict(dv=addr(6) + 2), dict(ws=addr(2)), dict(ws=addr(7))):
        assert attn(lib, **bad) == _lib.MI_ERR_ALIASING, bad
    # column blocks of one [rows, 3C] matrix may not overlap each other either
    assert attn(lib, dq=addr(5), dk=addr(5) + 128 * 2 - 2, dv=addr(5) + 512, lddq=384, lddk=384, lddv=384) == _lib.MI_ERR_ALIASING
    # ... nor the next batch's: the last row of dk (dv) of one batch in the first of dq (dq or dk) of the next
    joint = dict(dq=addr(5), dk=addr(5) + 256, dv=addr(5) + 512, lddq=384, lddk=384, lddv=384)
    for s in (63 * 384 + 128, 63 * 384 + 256, 64 * 384 - 1):
        assert attn(lib, **joint, sdq=s, sdk=s, sdv=s) == _lib.MI_ERR_ALIASING, s
    s = 63 * 384 + 128  # dq's own rows end before the next batch; dk's begin behind dq's of the next batch
    assert attn(lib, dq=addr(5), dk=addr(5) + 256, lddq=384, lddk=384, sdq=s, sdk=s) == _lib.MI_ERR_ALIASING
    assert attn(lib, dq=addr(5) + 256, dk=addr(5), lddq=384, lddk=384, sdq=s, sdk=s) == _lib.MI_ERR_ALIASING
    # of different lengths: the longer one's last row counts
    s = 64 * 384
    assert attn(lib, dq=addr(5) + 512, dk=addr(5), dv=addr(5) + 256, Tq=65, lddq=384, lddk=384, lddv=384, sdq=s, sdk=s, sdv=s) == _lib.MI_ERR_INVALID_ARG
    s = 64 * 384 + 128
    assert attn(lib, dq=addr(5), dk=addr(5) + 256, Tk=65, lddq=384, lddk=384, sdq=s, sdk=s) == _lib.MI_ERR_ALIASING
    # what fits gets past this check, to the workspace's
    for kw in (dict(), dict(sdq=64 * 384, sdk=64 * 384, sdv=64 * 384), dict(batch=1, sdq=1, sdk=1, sdv=1)):
        assert attn(lib, **{**joint, **kw}, ws=None) == _lib.MI_ERR_INVALID_ARG, kw
    assert ctypes.sizeof(_lib.MiAttnBwdArgs) == ctypes.sizeof(_lib.MiAttnArgs) + 4 * 8 + 8 * 8
