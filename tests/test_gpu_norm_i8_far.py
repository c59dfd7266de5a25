"""GroupNorm, the quantiser and the 8-bit product on tensors whose rows and images lie more than 4 GiB apart: the bits of the same data
packed."""
import numpy as np
import pytest

import norm_i8_ref as ref
from sdvk_amd import ops
from sdvk_amd.hip import DeviceBuffer, synchronize

pytestmark = pytest.mark.gpu

H = np.float16


@pytest.fixture(autouse=True)
def plans(gpu):
    ops.tuning_reset()


def spread(arr, ld):
    """[rows][cols] at a row stride of ld elements in a buffer of its own."""
    e = arr.itemsize
    b = DeviceBuffer(((arr.shape[0] - 1) * ld + arr.shape[1]) * e)
    for r, row in enumerate(arr):
        b.upload(row, offset=r * ld * e)
    return b


def gather(buf, rows, cols, ld, dt):
    e = np.dtype(dt).itemsize
    return np.stack([buf.download(dt, cols, offset=r * ld * e) for r in range(rows)])


@pytest.mark.parametrize("P,out", [(40, "f16"), (700, "f16"), (700, "i8"), (701, "f32")])
def test_images(gpu, P, out):
    """Two images, the second 4.3 GB behind the first, forward and backward (one launch and several; odd strides): the bits of the same
    images near each other."""
    print("[case] GroupNorm, image stride 2^31 + 64 elements", P, out, flush=True)
    odd = P == 701
    B, C, G = 2, 320, 32
    # the near images' stride takes the same kernels: those for 16-byte places, or those for any
    s, n = (1 << 31) + (63 if odd else 64), P * C + (63 if odd else 0)
    r = ref.rng_of(51)
    x, dy = (r.standard_normal((B, P * C)).astype(H) for _ in range(2))
    dt, code = {"f16": (H, ops.MI_F16), "i8": (np.int8, ops.MI_I8), "f32": (np.float32, ops.MI_F32)}[out]
    size = dict(batch=B, pixels=P, C=C, groups=G)
    kw = dict(x_dtype=ops.MI_F16, y_dtype=code, act=ops.MI_ACT_SILU, **size)
    ws = DeviceBuffer(ops.groupnorm_bwd_ws_bytes(**size))
    near, y, sc = spread(x, n), DeviceBuffer(B * n * 4), DeviceBuffer(B * P * 4)
    scale = dict(y_scale=sc) if out == "i8" else {}
    ops.groupnorm(near, None, None, y, ws, sx=n, sy=n, **scale, **kw)
    synchronize()
    want = gather(y, B, P * C, n, dt)
    assert np.any(want)
    far, fy = spread(x, s), DeviceBuffer((s + P * C) * np.dtype(dt).itemsize)
    ops.groupnorm(far, None, None, fy, ws, sx=s, sy=s, **scale, **kw)
    synchronize()
    assert np.array_equal(gather(fy, B, P * C, s, dt).view(np.uint8), want.view(np.uint8))
    if out == "i8":
        return
    bkw = dict(x_dtype=ops.MI_F16, dy_dtype=ops.MI_F16, act=ops.MI_ACT_SILU, **size)
    ndy, dx, dg, db = spread(dy, n), DeviceBuffer(B * n * 2), DeviceBuffer(C * 4), DeviceBuffer(C * 4)
    ops.groupnorm_bwd(near, None, None, ndy, dx, dg, db, ws, res=ndy, sx=n, sdy=n, sdx=n, sres=n, **bkw)
    synchronize()
    want = [gather(dx, B, P * C, n, H), dg.download(np.float32, C), db.download(np.float32, C)]
    fdy, fdx = spread(dy, s), DeviceBuffer((s + P * C) * 2)
    ops.groupnorm_bwd(far, None, None, fdy, fdx, dg, db, ws, res=fdy, sx=s, sdy=s, sdx=s, sres=s, **bkw)
    synchronize()
    got = [gather(fdx, B, P * C, s, H), dg.download(np.float32, C), db.download(np.float32, C)]
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(got, want))


@pytest.mark.parametrize("ld", [1 << 22, (1 << 22) + 16, (1 << 23) + 5])
def test_rows(gpu, ld):
    """Codes, activations and results in rows of 4 MB and more, the last ones past 4 GiB."""
    print("[case] product and quantiser, row stride", ld, flush=True)
    M, N, K = 1060, 70, 96
    r = ref.rng_of(52)
    x = r.standard_normal((M, K)).astype(H)
    w = r.integers(-127, 128, (N, K)).astype(np.int8)
    sw = DeviceBuffer.from_array(r.uniform(0.5, 2, N).astype(np.float32))
    W, near, q, sc, C = DeviceBuffer.from_array(w), DeviceBuffer.from_array(x), DeviceBuffer(M * K), DeviceBuffer(M * 4), DeviceBuffer(M * N * 4)
    ops.quantize_rows_i8(near, q, sc, M, K, dtype=ops.MI_F16)
    ops.gemm_nt_i8(q, sc, W, sw, C, M, N, K)
    synchronize()
    want = [q.download(np.int8, M * K).reshape(M, K), sc.download(np.float32, M), C.download(np.float32, M * N).reshape(M, N)]
    assert np.any(want[2])
    far, fq, fC = spread(x, ld), DeviceBuffer(M * ld), DeviceBuffer(M * ld * 4)
    ops.quantize_rows_i8(far, fq, sc, M, K, dtype=ops.MI_F16, ldx=ld, ldq=ld)
    ops.gemm_nt_i8(fq, sc, spread(w, ld), sw, fC, M, N, K, lda=ld, ldw=ld, ldc=ld)
    synchronize()
    got = [gather(fq, M, K, ld, np.int8), sc.download(np.float32, M), gather(fC, M, N, ld, np.float32)]
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(got, want))


def test_wide_results(gpu):
    """More than 2^32 bytes of results and 2^31 values of activations."""
    print("[case] product of 2^20 + 3 rows, quantiser of 2^21 + 5 rows", flush=True)
    M, N, K = (1 << 20) + 3, 1100, 16
    r = ref.rng_of(53)
    a, w = (r.integers(-127, 128, (n, K)).astype(np.int8) for n in (M, N))
    sa, sw = (r.uniform(0.5, 2, n).astype(np.float32) for n in (M, N))
    C = DeviceBuffer(M * N * 4)
    ops.gemm_nt_i8(DeviceBuffer.from_array(a), DeviceBuffer.from_array(sa), DeviceBuffer.from_array(w), DeviceBuffer.from_array(sw), C, M, N, K)
    synchronize()
    for m in (0, 1, M // 2, (1 << 32) // (N * 4), M - 1):
        got = C.download(np.float32, N, offset=m * N * 4)
        part = (a[m].astype(np.float64) @ w.astype(np.float64).T) * np.float64(sa[m]) * sw
        assert np.all(np.abs(got - part) <= 4 * ref.U * np.abs(part)), m
    rows, cols = (1 << 21) + 5, 1024
    row = (r.standard_normal(cols) * 3).astype(np.float32)
    x = DeviceBuffer(rows * cols * 4)
    x.fill_zero()
    for m in (0, rows // 2, rows - 1):
        x.upload(row, offset=m * cols * 4)
    q, sc = DeviceBuffer(rows * cols), DeviceBuffer(rows * 4)
    ops.quantize_rows_i8(x, q, sc, rows, cols)
    synchronize()
    want, ws = ref.codes_of(row[None])
    s = sc.download(np.float32, rows)
    assert np.count_nonzero(s == ws[0]) == 3 and np.count_nonzero(s == np.float32(2.0 ** -126)) == rows - 3
    for m in (0, rows // 2, rows - 1):
        assert np.array_equal(q.download(np.int8, cols, offset=m * cols), want[0])
    assert not np.any(q.download(np.int8, cols, offset=(rows - 2) * cols))


def test_many_columns(gpu):
    """Two rows and 2^27 columns: more of the few-row kernel's tiles than a launch has workgroups."""
    print("[case] product of 2 x (2^27 + 21)", flush=True)
    M, N, K = 2, (1 << 27) + 21, 16
    r = ref.rng_of(54)
    a, w = (r.integers(-127, 128, (n, K)).astype(np.int8) for n in (M, 3))
    sa = r.uniform(0.5, 2, M).astype(np.float32)
    W, C = DeviceBuffer(N * K), DeviceBuffer(M * N * 2)
    W.fill_zero()
    at = (0, N // 2, N - 1)
    for n, row in zip(at, w):
        W.upload(row, offset=n * K)
    ops.gemm_nt_i8(DeviceBuffer.from_array(a), DeviceBuffer.from_array(sa), W, DeviceBuffer.from_array(np.full(N, 0.0625, np.float32)), C, M, N, K, c_dtype=ops.MI_F16)
    synchronize()
    for m in range(M):
        for n, row in zip(at, w):
            part = (a[m].astype(np.float64) @ row.astype(np.float64)) * np.float64(sa[m]) * 0.0625
            assert abs(float(C.download(H, 1, offset=(m * N + n) * 2)[0]) - part) <= 2.0 ** -11 * abs(part) * 1.001, (m, n)
        assert not np.any(C.download(H, 1000, offset=(m * N + N // 2 + 1) * 2)) and not np.any(C.download(H, 1000, offset=(m * N + N - 1001) * 2))
