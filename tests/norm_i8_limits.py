"""GroupNorm, the token quantiser and the 8-bit product at the edges of what their documentation promises, against plain 64-bit formulas:
cases that run on any backend with the C-ABI (the GPU, or the CPU emulator of tests/kemu), with the bounds of tests/norm_i8_ref.py.
"""
from __future__ import annotations

import ctypes
from unittest import mock

import numpy as np

import norm_i8_ref
from bwd_ref import CODE, DT, SENTINEL, U, Arena, check, f64, rng_of
from norm_i8_ref import codes_of
from sdvk_amd._lib import MiGroupnormArgs

F127, R127 = np.float32(127), np.float32(1) / np.float32(127)


def reciprocal_codes(x):
    """What a scale of max|x| * (1 / 127) gives in place of the rounded quotient max|x| / 127."""
    scale = np.abs(x).max(1) * R127
    return np.rint(f64(x) / f64(scale)[:, None]).astype(np.int8), scale


def rows_reciprocal(rng, rows, cols, typ):
    """Rows whose maximum gives another scale by a product with 1 / 127, of values at the ties of the quotient's."""
    if typ == "f16":
        every = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16)
        every = every[every > 1e-3]
        tops = every[every > 1].astype(np.float32)
        tops = tops[tops / F127 != tops * R127]
        found = []
        for t in rng.permutation(tops):
            v = every[every.astype(np.float32) < t].astype(np.float32)
            q = [np.rint(f64(v) / float(s)) for s in (t / F127, t * R127)]
            if np.any(q[0] != q[1]):
                found.append((t, v[q[0] != q[1]]))
            if len(found) == rows:
                break
    else:
        tops = (2.0 ** rng.uniform(-10, 10, 64 * rows)).astype(np.float32)
        tops = tops[tops / F127 != tops * R127][:rows]
        found = []
        for t in tops:
            s = t / F127
            v = ((rng.integers(0, 127, 4 * cols) + 0.5) * float(s)).astype(np.float32)
            v = np.concatenate([v, np.nextafter(v, np.float32(0)), np.nextafter(v, t)])
            q = [np.rint(f64(v) / float(c)) for c in (s, t * R127)]
            found.append((t, v[q[0] != q[1]]))
    assert len(found) == rows and all(len(v) for _, v in found)
    x = np.stack([np.resize(v, cols) for _, v in found]) * rng.choice([-1, 1], (rows, cols))
    x[:, cols // 3] = [t for t, _ in found]
    return x


def rounded_half_codes(x):
    """The nearest codes where the rest of a product with 1 / scale is held against half a scale in fp32: of a scale below 2^-125 with an
    odd last place that half is no fp32 number, and rounds."""
    scale = np.abs(x).max(1) / F127
    inv, half = np.float32(1) / scale, np.float32(0.5) * scale
    t = np.rint(f64(x) * f64(inv)[:, None])
    r = (f64(x) - t * f64(scale)[:, None]).astype(np.float32)
    off = np.abs(r).view(np.uint32) + (t % 2 != 0) > half.view(np.uint32)[:, None]
    return (t + np.where(off, np.sign(r), 0)).astype(np.int8), scale


def rows_half(rng, rows, cols, typ):
    """Rows of the smallest scales above the floor (maxima of 1.5e-36 to 3e-36), of values a step of fp32 from a tie."""
    found = []
    while len(found) < rows:
        m = 2 * int(rng.integers(2 ** 22, 2 ** 23)) + 1  # the scale in steps of 2^-149
        t = np.float32(127 * m * 2.0 ** -149)
        s = t / F127
        if s != m * 2.0 ** -149:
            continue
        n = np.array([k * m + (m + o) // 2 for k in range(8) for o in (-1, 1)], np.float64)
        v = (n * 2.0 ** -149).astype(np.float32)
        v = v[f64(v) == n * 2.0 ** -149]
        x = np.concatenate([[t], v])[None].astype(np.float32)
        q = [c[0, 1:] for c, _ in (codes_of(x), rounded_half_codes(x))]
        if np.any(q[0] != q[1]):
            found.append((t, v[q[0] != q[1]]))
    x = np.stack([np.resize(v, cols) for _, v in found]) * rng.choice([-1, 1], (rows, cols))
    x[:, cols // 3] = [t for t, _ in found]
    return x


ROWS = {"reciprocal": (rows_reciprocal, reciprocal_codes), "half": (rows_half, rounded_half_codes)}


def rows_of(rng, rows, cols, typ, kind):
    """(x, codes and scales by the definition): the mistake that the rows are made for has other codes in each of them."""
    make, mistake = ROWS[kind]
    x = make(rng, rows, cols, typ).astype(DT[typ])
    right, wrong = codes_of(x.astype(np.float32)), mistake(x.astype(np.float32))
    assert np.all((right[0] != wrong[0]).any(1))
    return x, right


def codes(be, *, rows, cols, kind, typ="f32", N=24, seed=11):
    """The quantiser's codes and scales, and the product of them, of rows at a rounding's edge."""
    rng = rng_of(seed)
    x, (q, s) = rows_of(rng, rows, cols, typ, kind)
    A = Arena(be)
    bx = A.put(x.reshape(-1))
    bq, bs = A.out(rows * cols, np.int8), A.out(rows, np.float32)
    be.call("mi_quantize_rows_i8", bx.ptr, CODE[typ], bq.ptr, bs.ptr, rows, cols, 0, 0, None)
    got, gs = be.get(bq, np.int8, rows * cols).reshape(rows, cols), be.get(bs, np.float32, rows)
    assert np.array_equal(gs, s), np.flatnonzero(gs != s)[:5]
    assert np.array_equal(got, q), [(i, x[tuple(i)], s[i[0]], got[tuple(i)], q[tuple(i)]) for i in np.argwhere(got != q)[:5]]
    w = rng.integers(-127, 128, (N, cols)).astype(np.int8)
    sw = rng.uniform(0.5, 2, N).astype(np.float32)
    bw, bsw, bc = A.put(w.reshape(-1)), A.put(sw), A.out(rows * N, np.float32)
    be.call("mi_gemm_nt_i8", bq.ptr, bs.ptr, bw.ptr, bsw.ptr, None, bc.ptr, 0, rows, N, cols, 0, 0, 0, 0, None)
    want = f64(q) @ f64(w).T * f64(s)[:, None] * f64(sw)
    # float(sum), its product with the row's scale, the fma
    check(be.get(bc, np.float32, rows * N).reshape(rows, N), want, 4.01 * U * np.abs(want) + 1e-44, "linear")
    A.unchanged()


# ---------------------------------------------------------------- GroupNorm --

def pixels_of(kind):
    """Pixels in the place of norm_i8_ref.pixels_of's."""
    def make(rng, B, P, C, offset, outlier):
        if kind == "signs":  # magnitudes just below the documented 1e18
            return rng.choice([-9.99e17, 9.99e17], (B, P, C))
        if kind == "range":
            return rng.uniform(-9.99e17, 9.99e17, (B, P, C))
        if kind == "halves":  # the first row of a chunk and of a thread on one side, the rest on the other
            x = np.full((B, P, C), 9.99e17)
            x[:, ::2] = -9.99e17
            x[:, 0] = -9.99e17
            return x
        if kind == "ratio":  # a mean 1e5 times the spread
            return 1000 + 0.01 * rng.standard_normal((B, P, C))
        assert kind == "single"  # one value of a group
        x = np.zeros((B, P, C))
        x[:, 0, ::7] = 9.99e17
        return x
    return make


def norm(be, *, pixels, **case):
    """norm_i8_ref.groupnorm, or groupnorm_bwd (dtyp given), of other pixels."""
    with mock.patch.object(norm_i8_ref, "pixels_of", pixels_of(pixels)):
        (norm_i8_ref.groupnorm_bwd if "dtyp" in case else norm_i8_ref.groupnorm)(be, **case)


def outliers(be, *, C, G, typ, B=256, P=2048, first=1, every=3, seed=13):
    """The statistics of the first image of a batch whose images are a chunk each: a thread takes up to 2048 rows of its columns. The first
    rows of every third column are 1000 times the others' spread and more. (Images overlap in x, a row apart; on the emulator the first alone runs.)"""
    rng = rng_of(seed)
    x = rng.standard_normal((P + B - 1, C)) * 0.01
    size = 500.0 * 8 ** rng.random(G)
    x[:first, ::every] = np.repeat(size, C // G)[::every]
    x = x.astype(DT[typ])
    A = Arena(be)
    bx = A.put(x.reshape(-1))
    emulated = hasattr(be, "E")
    by = be.E.buf(nbytes=B * P * C * 2) if emulated else be.buf(np.zeros(B * P * C, np.float16))
    bst = A.out(B * G * 4, np.float32)
    need = be.value("mi_groupnorm_ws_bytes", B, P, C, G)
    ws = be.buf(np.full(need, 0xff, np.uint8))
    a = MiGroupnormArgs(bx.ptr, None, None, by.ptr, None, bst.ptr, B, P, C, G, CODE[typ], CODE["f16"], 0, 1e-5, C, C, C, P * C)
    if emulated:
        be.E.sample("gn_part_kernel|0|*|*;gn_apply_kernel|-1|*|*")
    be.call("mi_groupnorm", ctypes.byref(a), ws.ptr, need, None)
    if emulated:
        be.E.sample("")
    q = norm_i8_ref.Group(x[None, :P], G, 1e-5)
    st = f64(be.get(bst, np.float32, G * 4)).reshape(G, 4)
    # additions of up to 2048 squares to a sum that the outlier's makes up, and of 16 rows about the outlier itself (a sum 16 times as large)
    e_var = (P + 16 * 16 + 40) * U * q.var.reshape(G)
    e_mean = (P + 16 * 16 + 40) * U * np.sqrt(q.var.reshape(G))
    inv = q.inv.reshape(G)
    check(st[:, 0] + st[:, 1], q.mean.reshape(G), e_mean, "mean")
    check(st[:, 2], inv, inv * (0.5 * e_var / (q.var.reshape(G) + 1e-5) + 4 * U), "inv")
    A.unchanged()


def builds(be, *, M, N, K, out, mode=0, seed=14):
    """Every build of the product, storing whole runs or element by element, gives the same bits."""
    rng = rng_of(seed)
    a, w = (rng.integers(-127, 128, (r, K)).astype(np.int8) for r in (M, N))
    sa, sw = (rng.uniform(0.5, 2, M) / 128).astype(np.float32), (rng.uniform(0.5, 2, N) / 256).astype(np.float32)
    bias, dt = rng.standard_normal(N).astype(np.float32), DT[out]
    old = rng.standard_normal((M, N)).astype(dt)
    A = Arena(be)
    ba, bw, bsa, bsw, bb = (A.put(np.ascontiguousarray(t).reshape(-1)) for t in (a, w, sa, sw, bias))
    first = None
    for cfg in ("0", "2", "3", "4", "5", "6", "7", "8", None):
        for ldc in (N, N + 1):
            c = np.zeros((M, ldc), dt)
            c[:, :N] = old
            bc = A.out(0, dt, c.reshape(-1))
            be.tune("gemm_i8_cfg", cfg)
            be.call("mi_gemm_nt_i8", ba.ptr, bsa.ptr, bw.ptr, bsw.ptr, bb.ptr, bc.ptr, CODE[out], M, N, K, mode, 0, 0, ldc, None)
            be.tune("gemm_i8_cfg", None)
            got = be.get(bc, dt, M * ldc).reshape(M, ldc)[:, :N]
            first = got if first is None else first
            bad = np.argwhere(got != first)
            assert not len(bad), (cfg, ldc, len(bad), [(tuple(map(int, i)), got[tuple(i)], first[tuple(i)]) for i in bad[:3]])
    A.unchanged()


def plain(be, *, of, **case):
    norm_i8_ref.OPS[of](be, **case)


OPS = {"codes": codes, "builds": builds, "norm": norm, "outliers": outliers, "plain": plain, "strided": plain}

# what takes a group in registers (units of four and two values, whole and part full), chunks, and element by element
NORM_SIZES = [dict(P=50, C=32, G=4), dict(P=256, C=64, G=1), dict(P=100, C=60, G=10, gap=2), dict(P=300, C=40, G=1), dict(P=600, C=320, G=32), dict(P=600, C=128, G=2), dict(P=300, C=33, G=1)]

CASES = {
    # a chunk's first value far from its mean, which many values make
    "plain": [dict(of="groupnorm", B=9, P=3, C=4096, G=1, offset=-20.0, outlier=300.0), dict(of="groupnorm", B=9, P=4, C=4096, G=1, outlier=5000.0, out="f16"), dict(of="groupnorm", B=2, P=14, C=2048, G=2, offset=-20.0, outlier=1000.0), dict(of="groupnorm", P=250, C=128, G=1, offset=3.0, outlier=3e4),
              dict(of="groupnorm", P=60, C=4096, G=1, offset=-20.0, outlier=300.0, out="f16"), dict(of="groupnorm", P=700, C=33, G=1, offset=-20.0, outlier=300.0), dict(of="groupnorm_bwd", P=3, C=4096, G=1, offset=-20.0)],
    "builds": [dict(M=70, N=64, K=48, out="f16"), dict(M=70, N=64, K=48, out="f16", mode=2), dict(M=33, N=136, K=16, out="f32")],
    "outliers": [dict(C=2048, G=16, typ="f32"), dict(C=2048, G=32, typ="f16"), dict(C=2048, G=16, typ="f32", first=5), dict(C=1024, G=8, typ="f16", first=64, every=1)],
    "norm": [dict(pixels=k, **c) for k in ("signs", "range", "halves", "single") for c in NORM_SIZES]
    + [dict(pixels="signs", P=40, C=320, G=32, out="i8"), dict(pixels="halves", P=300, C=64, G=2, out="i8", act=1), dict(pixels="signs", P=30, C=33, G=3, out="i8"), dict(pixels="range", B=2, P=513, C=64, G=1, out="f16", act=1)]
    + [dict(pixels=k, dtyp="f32", act=a, **c) for k, a in (("signs", 0), ("halves", 1)) for c in NORM_SIZES]
    + [dict(pixels="ratio", **o, **c) for o in (dict(act=1), dict(dtyp="f32")) for c in NORM_SIZES] + [dict(pixels="ratio", P=300, C=64, G=8, out="i8"), dict(pixels="ratio", P=50, C=64, G=8, out="i8", act=1)],
    "codes": [dict(rows=9, cols=64, kind="reciprocal"), dict(rows=20, cols=77, kind="reciprocal"), dict(rows=5, cols=2048, kind="reciprocal"), dict(rows=3, cols=1280, kind="reciprocal", typ="f16"),
              dict(rows=40, cols=64, kind="half"), dict(rows=9, cols=75, kind="half"), dict(rows=5, cols=2048, kind="half")],
}
GPU_CASES = {
    "builds": [dict(M=1024, N=1000, K=64, out="f16"), dict(M=1024, N=1000, K=64, out="f16", mode=2), dict(M=1024, N=1000, K=64, out="f16", mode=1), dict(M=1024, N=1000, K=64, out="f32", mode=2)],
    # more than 2^20 units of the kernels that stride
    "strided": [dict(of="groupnorm", B=32769, P=1, C=96, G=32, gap=1), dict(of="groupnorm", P=4194305, C=3, G=1), dict(of="groupnorm_bwd", B=32769, P=1, C=96, G=32, gap=1, act=1),
                dict(of="groupnorm_bwd", P=4194305, C=3, G=1), dict(of="quantize", rows=4194305, cols=3), dict(of="product", M=(1 << 26) + 1, N=1, K=1)],
    # chunks of 2048 rows; a workgroup's registers full
    "norm": [dict(pixels=k, **c) for k in ("signs", "halves") for c in (dict(B=256, P=2048, C=64, G=2), dict(P=20000, C=256, G=2, act=1), dict(P=1024, C=1280, G=32, out="i8"), dict(P=32768, C=4, G=4))]
    + [dict(pixels="ratio", P=20000, C=256, G=32), dict(pixels="ratio", P=1024, C=1280, G=32, dtyp="f32", act=1)]
    + [dict(pixels="signs", P=1024, C=1280, G=32, dtyp="f32"), dict(pixels="halves", B=256, P=2048, C=64, G=2, dtyp="f32")],
    "codes": [dict(rows=154, cols=2048, kind="reciprocal", N=1280), dict(rows=16, cols=5120, kind="reciprocal", typ="f16", N=640), dict(rows=300, cols=1280, kind="half")],
}
