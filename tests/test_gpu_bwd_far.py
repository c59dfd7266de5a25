"""Backward operators on tensors whose rows and batches lie more than 4 GiB apart: the bits of the same data packed."""
import numpy as np
import pytest

import bwd_ref
from sdvk_amd import ops
from sdvk_amd.hip import DeviceBuffer, synchronize

pytestmark = pytest.mark.gpu

H = np.float16


@pytest.fixture(autouse=True)
def plans(gpu):
    ops.tuning_reset()


def test_attention_batches(gpu):
    """fp16 inputs in one allocation, the second batch 4.3 GB behind the first; gradients far apart too."""
    print("[case] attention, batch stride 2^31 + 64 elements", flush=True)
    B, T, C, heads, s = 2, 150, 128, 2, (1 << 31) + 64
    r = bwd_ref.rng_of(41)
    x = [(r.standard_normal((B, T, C)) * f).astype(H) for f in (1, 1, 1, 1, 0.1)]
    ws = DeviceBuffer(ops.fused_attention_bwd_ws_bytes(batch=B, Tq=T, Tk=T, C=C, heads=heads, dtype=ops.MI_F16))
    near = [DeviceBuffer.from_array(a.reshape(-1)) for a in x]
    out = [DeviceBuffer.from_array(np.full(B * T * C, 7, H)) for _ in range(3)]
    kw = dict(batch=B, Tq=T, Tk=T, C=C, heads=heads, dtype=ops.MI_F16)
    ops.fused_attention_bwd(*near, *out, ws, **kw)
    synchronize()
    want = [b.download(H, B * T * C).reshape(B, T, C) for b in out]
    assert all(np.all(np.isfinite(w)) and np.any(w) for w in want)

    step = T * C * 2
    far = DeviceBuffer((s * 2) + 5 * step)
    for i, a in enumerate(x):
        for b in range(B):
            far.upload(a[b].reshape(-1), offset=i * step + b * s * 2)
    grads = DeviceBuffer(s * 2 + step)
    small = [DeviceBuffer.from_array(np.full(B * T * C, 7, H)) for _ in range(2)]
    strides = dict(sq=s, sk=s, sv=s, so=s, sdout=s)
    for n in range(3):  # each gradient far apart once
        d = [small[0], small[1]]
        d.insert(n, grads)
        ops.fused_attention_bwd(*(far.value + i * step for i in range(5)), *d, ws, **kw, **strides, **{"sd" + "qkv"[n]: s})
        synchronize()
        for b in range(B):
            got = grads.download(H, T * C, offset=b * s * 2).reshape(T, C)
            assert np.array_equal(got.view(np.uint16), want[n][b].view(np.uint16)), ("qkv"[n], b)


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_linear_rows(gpu, typ):
    """Rows of dC and dA a few MB apart, the last ones past 4 GiB."""
    print(f"[case] linear {typ}, row strides of 2^21 elements and more", flush=True)
    dt, code = bwd_ref.DT[typ], bwd_ref.CODE[typ]
    e = np.dtype(dt).itemsize
    ld = (1 << 22) // e * 2 - 8
    M, N, K = (1 << 32) // (ld * e) + 40, 72, 96
    r = bwd_ref.rng_of(42)
    c = (r.standard_normal((M, N)) * 0.1).astype(dt)
    raw, _ = bwd_ref.q8_blocks(r.standard_normal((N, K)) * 0.05)
    W, near = DeviceBuffer.from_array(raw), DeviceBuffer.from_array(c.reshape(-1))
    out = DeviceBuffer.from_array(np.full(M * K, 7, dt))
    ops.gemm_nt_q8_0_bwd(near, W, out, M, N, K, dtype=code)
    synchronize()
    want = out.download(dt, M * K).reshape(M, K)
    assert np.all(np.isfinite(want)) and np.any(want)
    far, res = DeviceBuffer(M * ld * e), DeviceBuffer(M * ld * e)
    for m in range(M):
        far.upload(c[m], offset=m * ld * e)
    ops.gemm_nt_q8_0_bwd(far, W, res, M, N, K, dtype=code, ldc=ld, lda=ld)
    synchronize()
    got = np.stack([res.download(dt, K, offset=m * ld * e) for m in range(M)])
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))


def test_geglu_gemm_rows(gpu):
    """Rows of dG and dH a few MB apart, the last ones past 4 GiB."""
    print("[case] geglu_gemm, row strides of 2^21 - 8 elements", flush=True)
    ld, F, K = (1 << 21) - 8, 40, 64
    M = (1 << 32) // (ld * 2) + 40
    r = bwd_ref.rng_of(43)
    a, g = r.standard_normal((M, K)).astype(H), (r.standard_normal((M, F)) * 0.1).astype(H)
    raw, _ = bwd_ref.q8_blocks(r.standard_normal((2 * F, K)) * 0.05)
    A, W, near = DeviceBuffer.from_array(a.reshape(-1)), DeviceBuffer.from_array(raw), DeviceBuffer.from_array(g.reshape(-1))
    out = DeviceBuffer.from_array(np.full(M * 2 * F, 7, H))
    ops.gemm_nt_q8_0_geglu_bwd(A, W, near, out, M, F, K)
    synchronize()
    want = out.download(H, M * 2 * F).reshape(M, 2 * F)
    assert np.all(np.isfinite(want)) and np.any(want)
    far, res = DeviceBuffer(M * ld * 2), DeviceBuffer(M * ld * 2)
    for m in range(M):
        far.upload(g[m], offset=m * ld * 2)
    ops.gemm_nt_q8_0_geglu_bwd(A, W, far, res, M, F, K, lddg=ld, lddh=ld)
    synchronize()
    got = np.stack([res.download(H, 2 * F, offset=m * ld * 2) for m in range(M)])
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


def test_layernorm_columns(gpu):
    """More columns than a launch has threads for at 32 columns a workgroup of 1024. Signs that alternate every 64 (x) and
    every 128 columns (dy): every sum over columns is exact, mean(dy) = mean(dy xh) = 0, and what is left is the rounding of
    1 / sqrt(var + eps), three operations, and of the products."""
    d = (1 << 26) + 256
    print(f"[case] LayerNorm of {d} columns", flush=True)
    s = np.where(np.arange(d) // 64 % 2 == 0, 1, -1).astype(np.float32)
    t = np.where(np.arange(d) // 128 % 2 == 0, 1, -1).astype(np.float32)
    a, b = np.float32([1, 2]), np.float32([3, 0.5])
    x, dy = (DeviceBuffer.from_array((f[:, None] * v).reshape(-1)) for f, v in ((a, s), (b, t)))
    ws = DeviceBuffer(ops.layernorm_bwd_ws_bytes(2, d))
    dx, dg, db = (DeviceBuffer.from_array(np.full(n * d, 7, np.float32)) for n in (2, 1, 1))
    ops.layernorm_bwd(x, None, dy, dx, dg, db, ws, 2, d)
    synchronize()
    inv = 1 / np.sqrt(np.float64(a) ** 2 + np.float64(np.float32(1e-5)))
    tol = 8 * bwd_ref.U
    got = dx.download(np.float32, 2 * d).reshape(2, d)
    for r in range(2):
        assert np.max(np.abs(got[r] - (inv[r] * b[r]) * t)) <= tol * inv[r] * b[r], r
    want = float((a * b * inv).sum())
    assert np.max(np.abs(dg.download(np.float32, d) - want * (s * t))) <= tol * want
    assert np.array_equal(db.download(np.float32, d), 3.5 * t)
    ops.layernorm_bwd(x, None, dy, dx, dg, db, ws, 0, d)
    synchronize()
    assert not dg.download(np.float32, d).any() and not db.download(np.float32, d).any()


def test_linear_columns(gpu):
    """One row and more 32-wide blocks of columns than a launch has workgroups of 1024 threads: a weight of one row whose
    quants count through -127 .. 127, its scales powers of two, so that every product is exact."""
    K = (1 << 27) + 64
    print(f"[case] linear of {K} columns, one row", flush=True)
    q = (np.arange(K) % 255 - 127).astype(np.int8).reshape(-1, 32)
    d = np.float16(2.0) ** (np.arange(K // 32) % 7 - 3).astype(np.float16)
    W = DeviceBuffer.from_array(np.concatenate([d[:, None].view(np.uint8), q.view(np.uint8)], 1).reshape(-1))
    dC, dA = DeviceBuffer.from_array(np.float32([3.0])), DeviceBuffer.from_array(np.full(K, 7, np.float32))
    ops.gemm_nt_q8_0_bwd(dC, W, dA, 1, 1, K)
    synchronize()
    want = 3 * q.astype(np.float32) * d.astype(np.float32)[:, None]
    assert np.array_equal(dA.download(np.float32, K), want.reshape(-1))
