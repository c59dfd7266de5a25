"""GroupNorm, the token quantiser and the 8-bit product against plain 64-bit formulas: cases that run on any backend with the
C-ABI (the GPU, or the CPU emulator of tests/kemu), with error bounds derived from the operators' roundings.

u = 2^-24 is half a step of fp32, h = 2^-11 half a step of fp16, both relative to the value.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from bwd_ref import CODE, DT, SENTINEL, Arena, U, check, f64, rng_of, store_err
from sdvk_amd._lib import MiGroupnormArgs, MiGroupnormBwdArgs

I8 = 2
SILU = 1


def place(rng_values, ld, s, off, C):
    """A flat buffer of [batch][pixels][C] values at row stride ld, image stride s, `off` elements in; gaps of SENTINEL."""
    B, P, _ = rng_values.shape
    n = off + ((B - 1) * s + (P - 1) * ld + C if B and P else 0)
    buf = np.full(max(n, 1), SENTINEL, dtype=rng_values.dtype)
    view(buf, off, B, P, C, ld, s)[...] = rng_values
    return buf


def view(flat, off, B, P, C, ld, s):
    e = flat.itemsize
    return np.lib.stride_tricks.as_strided(flat[off:], (B, P, C), (s * e, ld * e, e))


def outside(flat, off, B, P, C, ld, s):
    rest = np.ones(flat.shape, dtype=bool)
    view(rest, off, B, P, C, ld, s)[...] = False
    return flat[rest]


def strides(order, B, P, C, gap):
    """(row stride, image stride): images one after another, or the images' rows in turn."""
    return (C + gap, P * (C + gap) + gap) if order == "images" else (B * (C + gap), C + gap)


def pixels_of(rng, B, P, C, offset, outlier):
    x = rng.standard_normal((B, P, C)) * (0.5 + np.abs(rng.standard_normal(C))) + rng.standard_normal(C) + offset
    if outlier:
        x[:, 0, 0] = outlier
        x[:, P // 2, C // 2] = -outlier
    return x


class Group:
    """The 64-bit statistics of x, and bounds of what the kernels' differ by."""

    def __init__(self, x, G, eps):
        B, P, C = x.shape
        cg = C // G
        X = f64(x).reshape(B, P, G, cg)
        self.n = P * cg
        self.mean = X.mean((1, 3), keepdims=True)
        self.xc = X - self.mean
        self.var = (self.xc ** 2).mean((1, 3), keepdims=True)
        e = float(np.float32(eps))
        self.inv = 1 / np.sqrt(self.var + e)
        self.xh = self.xc * self.inv
        # a chunk's shift lies among its rows' means (of a group); sums about it: chains of up to 2048 rows, in fact
        # P / rows-at-a-time of them, and a tree over the workgroup; fp32 values of the differences
        off2 = (X.mean(3, keepdims=True) - self.mean) ** 2
        far = self.var + off2.max(1, keepdims=True, initial=0)
        chain = min(P, 2048) + 16 + 12
        self.e_mean = chain * U * np.sqrt(far)
        self.e_var = 2 * chain * U * far + self.e_mean ** 2
        with np.errstate(invalid="ignore", divide="ignore"):
            self.e_inv = np.where(self.var + e > 0, self.inv * (0.5 * self.e_var / (self.var + e) + 3 * U), 0.0)
        # x - mean rounded, the mean's error, inv's
        self.e_xh = self.inv * (self.e_mean + U * np.abs(self.xc)) + np.abs(self.xc) * self.e_inv + 2 * U * np.abs(self.xh)


def silu_parts(z):
    s = 1 / (1 + np.exp(-np.clip(z, -700, 700)))
    return s, z * s, s * (1 + z * (1 / (1 + np.exp(np.clip(z, -700, 700)))))


def forward64(q, gamma, beta, act, shape):
    """(y, bound of y's error before it is stored)."""
    G, cg = q.xh.shape[2:]
    g, b = f64(gamma).reshape(1, 1, G, cg), f64(beta).reshape(1, 1, G, cg)
    z = q.xh * g + b
    e = np.abs(g) * q.e_xh + U * (3 * np.abs(q.xh * g) + 2 * np.abs(b) + np.abs(z))
    if act:
        _, y, _ = silu_parts(z)
        e = 1.1 * e + np.abs(y) * (2 * np.abs(z) + 8) * U + np.abs(z) * 2.0 ** -126
        z = y
    return z.reshape(shape), e.reshape(shape) + 1e-37


def affine_of(rng, C, kind):
    gamma = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32)
    beta = (0.3 * rng.standard_normal(C)).astype(np.float32)
    return (gamma if kind in ("both", "gamma") else None, beta if kind in ("both", "beta") else None)


def groupnorm(be, *, B=1, P, C, G, typ="f32", out="f32", act=0, affine="both", order="images", gap=0, ygap=0, off=0, yoff=0, offset=0.5,
              outlier=0.0, scale=1.0, eps=1e-5, keep=True, constant=False, seed=1):
    rng = rng_of(seed)
    x = (pixels_of(rng, B, P, C, offset, outlier) * scale).astype(DT[typ])
    if constant:
        x[...] = x[:1, :1, :1]
    gamma, beta = affine_of(rng, C, affine)
    ldx, sx = strides(order, B, P, C, gap)
    ldy, sy = strides(order, B, P, C, ygap)
    A = Arena(be)
    bx = A.put(place(x, ldx, sx, off, C))
    bg, bb = (A.put(t) if t is not None else None for t in (gamma, beta))
    odt = {"f32": np.float32, "f16": np.float16, "i8": np.int8}[out]
    ny = yoff + (B - 1) * sy + (P - 1) * ldy + C
    by = A.out(ny, odt)
    bs = A.out(B * P, np.float32) if out == "i8" else None
    bst = A.out(B * G * 4, np.float32) if keep else None
    need = be.value("mi_groupnorm_ws_bytes", B, P, C, G)
    assert need > 0
    ws = be.buf(np.full(need, 0xff, np.uint8))
    esz, osz = x.itemsize, np.dtype(odt).itemsize
    a = MiGroupnormArgs(be.at(bx, off * esz), bg.ptr if bg else None, bb.ptr if bb else None, be.at(by, yoff * osz), bs.ptr if bs else None,
                        bst.ptr if bst else None, B, P, C, G, CODE[typ], {"f32": 0, "f16": 1, "i8": I8}[out], act, eps,
                        0 if (gap == 0 and order == "images") else ldx, 0 if (ygap == 0 and order == "images") else ldy,
                        0 if (gap == 0 and order == "images") else sx, 0 if (ygap == 0 and order == "images") else sy)
    be.call("mi_groupnorm", ctypes.byref(a), ws.ptr, need, None)
    flat = be.get(by, odt, ny)
    got = view(flat, yoff, B, P, C, ldy, sy).copy()
    assert np.all(outside(flat, yoff, B, P, C, ldy, sy) == np.array(SENTINEL).astype(odt)), "wrote outside y"
    q = Group(x, G, eps)
    want, e = forward64(q, gamma if gamma is not None else np.ones(C), beta if beta is not None else np.zeros(C), act, (B, P, C))
    if out == "i8":
        sc = f64(be.get(bs, np.float32, B * P)).reshape(B, P, 1)
        top = np.abs(want).max(2, keepdims=True)
        s0 = np.maximum(top / 127, 2.0 ** -126)
        es = e.max(2, keepdims=True) / 127 + s0 * U
        check(sc, s0, es * 1.001, "groupnorm scale")
        assert np.abs(got.astype(int)).max() <= 127
        check(f64(got) * sc, want, 0.5 * sc * (1 + 1e-6) + e, "groupnorm codes")
        assert np.all((np.abs(got.astype(int)).max(2) == 127) | (top[..., 0] < 127 * 2.0 ** -126 * 1.01) | (e.max(2) > 0.1 * s0[..., 0])), "a row does not reach 127"
    else:
        check(got, want, e + store_err(want, out) * 1.01, "groupnorm y")
    if keep:
        st = f64(be.get(bst, np.float32, B * G * 4)).reshape(B, 1, G, 1, 4)
        check(st[..., 0] + st[..., 1], q.mean, q.e_mean + 2.0 ** -46 * np.abs(q.mean) + 1e-44, "groupnorm mean")
        check(st[..., 2], q.inv, q.e_inv + U * q.inv, "groupnorm inv")
        assert np.all(st[..., 3] == 0)
    A.unchanged()
    again = be.get(bs, np.float32, B * P) if bs else None
    be.call("mi_groupnorm", ctypes.byref(a), ws.ptr, need, None)
    assert np.array_equal(be.get(by, odt, ny).view(np.uint8), flat.view(np.uint8)), "a second call gave other bits"
    if bs:
        assert np.array_equal(be.get(bs, np.float32, B * P), again)


def backward64(q, dy, gamma, beta, act, res):
    """(dx, dgamma, dbeta) and bounds of their errors before they are stored."""
    B, P, G, cg = q.xh.shape
    g, b = f64(gamma).reshape(1, 1, G, cg), f64(beta).reshape(1, 1, G, cg)
    Y = f64(dy).reshape(q.xh.shape)
    W, eW = Y, np.zeros_like(Y)
    if act:
        z = q.xh * g + b
        ez = np.abs(g) * q.e_xh + U * (2 * np.abs(q.xh * g) + np.abs(b) + np.abs(z))
        s, _, sl = silu_parts(z)
        # |act''| <= 0.5; sigma is off by 5 u and by 2 u |z| of its complement, so is e sigma
        e_s = s * (5 + 2 * np.abs(z) * (1 - s)) * U
        rest = 1 - s
        e_r = rest * (7 + 4 * np.abs(z)) * U + 2.0 ** -125
        W = Y * sl
        eW = np.abs(Y) * (0.5 * ez + e_s * np.abs(1 + z * rest) + s * (np.abs(z) * e_r + U * (1 + np.abs(z * rest))) + 2 * U * np.abs(sl))
    n = q.n
    V, eV = W * g, np.abs(g) * eW + U * np.abs(W * g)
    chain = min(P, 2048) + 40
    m1, m2 = V.mean((1, 3), keepdims=True), (V * q.xh).mean((1, 3), keepdims=True)
    em1 = (chain * U * np.abs(V) + eV).mean((1, 3), keepdims=True) + U * np.abs(m1)
    em2 = (chain * U * np.abs(V * q.xh) + eV * np.abs(q.xh) + np.abs(V) * q.e_xh).mean((1, 3), keepdims=True) + U * np.abs(m2)
    body = V - m1 - q.xh * m2
    e_body = eV + em1 + np.abs(q.xh) * em2 + q.e_xh * np.abs(m2) + 2 * U * (np.abs(V) + np.abs(m1) + np.abs(q.xh * m2))
    dx = q.inv * body
    e_dx = q.inv * e_body + q.e_inv * np.abs(body) + U * np.abs(dx)
    shape = (B, P, G * cg)
    dx, e_dx = dx.reshape(shape), e_dx.reshape(shape)
    if res is not None:
        dx = dx + f64(res)
        e_dx = e_dx + U * np.abs(dx)
    t = W * q.xh
    dg = t.sum((0, 1)).reshape(-1)
    e_dg = (np.abs(W) * q.e_xh + eW * np.abs(q.xh) + chain * U * np.abs(t)).sum((0, 1)).reshape(-1)
    db = W.sum((0, 1)).reshape(-1)
    e_db = (eW + chain * U * np.abs(W)).sum((0, 1)).reshape(-1)
    return (dx, e_dx + 1e-37), (dg, e_dg + U * np.abs(dg) + 1e-37), (db, e_db + U * np.abs(db) + 1e-37)


def stats64(q):
    """What the forward pass keeps, rounded from 64 bits."""
    m = q.mean[:, 0, :, 0]
    hi = m.astype(np.float32)
    return np.stack([hi, (m - hi).astype(np.float32), q.inv[:, 0, :, 0].astype(np.float32), np.zeros_like(hi)], -1)


def groupnorm_bwd(be, *, B=1, P, C, G, typ="f32", dtyp="f32", act=0, affine="both", order="images", gap=0, dgap=0, off=0, doff=0, offset=0.5,
                  res=False, in_place=False, kept=False, weights=True, eps=1e-5, gstd=1.0, seed=2):
    rng = rng_of(seed)
    x = pixels_of(rng, B, P, C, offset, 0.0).astype(DT[typ])
    dy = (rng.standard_normal((B, P, C)) * gstd).astype(DT[dtyp])
    rs = (rng.standard_normal((B, P, C)) * gstd).astype(DT[typ]) if res or in_place else None
    gamma, beta = affine_of(rng, C, affine)
    ldx, sx = strides(order, B, P, C, gap)
    ldd, sd = strides(order, B, P, C, dgap)
    q = Group(x, G, eps)
    A = Arena(be)
    bx, bd = A.put(place(x, ldx, sx, off, C)), A.put(place(dy, ldd, sd, doff, C))
    bg, bb = (A.put(t) if t is not None else None for t in (gamma, beta))
    bst = A.put(stats64(q).reshape(-1)) if kept else None
    ndx = doff + (B - 1) * sd + (P - 1) * ldd + C
    bo = A.out(ndx, DT[typ], place(rs, ldd, sd, doff, C) if in_place else None)
    br = bo if in_place else A.put(place(rs, ldd, sd, doff, C)) if res else None
    bdg, bdb = A.out(C, np.float32), A.out(C, np.float32)
    need = be.value("mi_groupnorm_bwd_ws_bytes", B, P, C, G)
    ws = be.buf(np.full(need, 0xff, np.uint8))
    ex, ed = x.itemsize, dy.itemsize
    f = MiGroupnormArgs(be.at(bx, off * ex), bg.ptr if bg else None, bb.ptr if bb else None, None, None, bst.ptr if bst else None, B, P, C, G,
                        CODE[typ], CODE[dtyp], act, eps, ldx, 0, sx, 0)
    a = MiGroupnormBwdArgs(f, be.at(bd, doff * ed), be.at(br, doff * ex) if br else None, be.at(bo, doff * ex),
                           bdg.ptr if weights else None, bdb.ptr if weights else None, ldd, ldd, ldd, sd, sd, sd)
    be.call("mi_groupnorm_bwd", ctypes.byref(a), ws.ptr, need, None)
    (dx, e_dx), (dg, e_dg), (db, e_db) = backward64(q, dy, gamma if gamma is not None else np.ones(C), beta if beta is not None else np.zeros(C),
                                                   act, rs)
    flat = be.get(bo, DT[typ], ndx)
    assert np.all(outside(flat, doff, B, P, C, ldd, sd) == np.array(SENTINEL).astype(DT[typ])), "wrote outside dx"
    check(view(flat, doff, B, P, C, ldd, sd), dx, e_dx + store_err(dx, typ) * 1.01, "groupnorm dx")
    g1, g2 = be.get(bdg, np.float32, C), be.get(bdb, np.float32, C)
    if weights:
        check(g1, dg, e_dg, "groupnorm dgamma")
        check(g2, db, e_db, "groupnorm dbeta")
    else:
        assert np.all(g1 == np.float32(SENTINEL)) and np.all(g2 == np.float32(SENTINEL))
    A.unchanged()
    if not in_place:
        be.call("mi_groupnorm_bwd", ctypes.byref(a), ws.ptr, need, None)
        assert np.array_equal(be.get(bo, DT[typ], ndx).view(np.uint8), flat.view(np.uint8)), "a second call gave other bits"
        assert np.array_equal(be.get(bdg, np.float32, C), g1) and np.array_equal(be.get(bdb, np.float32, C), g2)


# --------------------------------------------------------------- 8-bit rows --

def codes_of(x):
    """(codes, scales) by the definition: the scale an fp32 number, the quotient exact (64 bits tell every pair of fp32
    numbers' quotient from a tie)."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(x).max(1)
        bad = ~np.isfinite(top)
        scale = np.maximum(top, np.float32(127 * 2.0 ** -126)) / np.float32(127)
        q = np.rint(f64(x) / f64(scale)[:, None])
    q[bad] = 0
    scale[bad] = np.nan
    return q.astype(np.int8), scale


def rows_with(rng, rows, cols, kind):
    x = rng.standard_normal((rows, cols))
    if kind == "ties":  # codes and halves of them, of scales that are short numbers
        x = rng.integers(-254, 255, (rows, cols)) * 0.5
        x[:, 0] = 127
        x *= rng.choice([1.0, 3.0, 0.375, 5 * 2.0 ** -20], (rows, 1))
    elif kind == "near":  # a step of fp32 off a tie
        k = rng.integers(-127, 127, (rows, cols)) + 0.5
        s = np.float32(1.0) + np.float32(2.0 ** -13) * rng.integers(0, 8000, (rows, 1))
        x = np.nextafter((k * s).astype(np.float32), np.float32(rng.choice([-1e9, 1e9]))).astype(np.float64)
        x[:, :1] = 127 * s
    elif kind == "sizes":  # from rows of zeros to the largest numbers
        x *= 10.0 ** np.resize(np.array([-45.0, -41, -39, -37.5, -20, 0, 20, 37.5]), rows)[:, None]
        x[::9] = 0
    elif kind == "broken":
        x[1 % rows, cols // 2] = np.inf
        x[2 % rows, 0] = np.nan
        x[3 % rows, cols - 1] = -np.inf
    return x


def quantize(be, *, rows, cols, typ="f32", kind="normal", ldx=0, ldq=0, off=0, qoff=0, seed=3):
    rng = rng_of(seed)
    with np.errstate(over="ignore"):
        x = rows_with(rng, rows, cols, kind).astype(np.float32).astype(DT[typ])
    lx, lq = ldx or cols, ldq or cols
    A = Arena(be)
    buf = place(x[None], lx, 0, off, cols)
    bx = A.put(buf)
    nq = qoff + (rows - 1) * lq + cols
    bq, bs = A.out(nq, np.int8), A.out(rows, np.float32)
    be.call("mi_quantize_rows_i8", be.at(bx, off * x.itemsize), CODE[typ], be.at(bq, qoff), bs.ptr, rows, cols, ldx, ldq, None)
    flat = be.get(bq, np.int8, nq)
    assert np.all(outside(flat, qoff, 1, rows, cols, lq, 0) == np.int8(SENTINEL)), "wrote outside q"
    q, s = codes_of(x.astype(np.float32))
    gs = be.get(bs, np.float32, rows)
    assert np.array_equal(gs, s, equal_nan=True), np.flatnonzero(gs != s)[:5]
    got = view(flat, qoff, 1, rows, cols, lq, 0)[0]
    assert np.array_equal(got, q), [(i, x[tuple(i)], s[i[0]], got[tuple(i)], q[tuple(i)]) for i in np.argwhere(got != q)[:5]]
    A.unchanged()


def product(be, *, M, N, K, out="f32", mode=0, bias=True, lda=0, ldw=0, ldc=0, off=0, woff=0, coff=0, extreme=False, broken=False, cfg=None, seed=4):
    rng = rng_of(seed)
    lo = -128 if extreme else -127
    a, w = (rng.integers(lo, 128, (r, K)).astype(np.int8) for r in (M, N))
    if extreme:
        a[0], w[0] = -128, -128
        a[-1], w[-1] = 127, -128
    sa = (10.0 ** rng.uniform(-6, 2, M)).astype(np.float32)
    sw = (10.0 ** rng.uniform(-6, 2, N)).astype(np.float32)
    if out == "f16":  # within fp16's range
        sa, sw = (rng.uniform(0.5, 2, M) / 128).astype(np.float32), (rng.uniform(0.5, 2, N) / (128 * max(1, math.sqrt(K)))).astype(np.float32)
    if broken:
        sa[M // 2] = np.nan
        a[M // 2] = 0
    b = rng.standard_normal(N).astype(np.float32)
    la, lw, lc = lda or K, ldw or K, ldc or N
    dt = DT[out]
    A = Arena(be)
    ba, bw = A.put(place(a[None], la, 0, off, K)), A.put(place(w[None], lw, 0, woff, K))
    bsa, bsw, bb = A.put(sa), A.put(sw), A.put(b)
    nc = coff + (M - 1) * lc + N
    init = np.full(nc, SENTINEL, dt)
    old = rng.standard_normal((M, N)).astype(dt)
    if mode:
        view(init, coff, 1, M, N, lc, 0)[0] = old
    bc = A.out(0, dt, init.copy())
    if cfg:
        be.tune("gemm_i8_cfg", cfg)
    be.call("mi_gemm_nt_i8", be.at(ba, off), bsa.ptr, be.at(bw, woff), bsw.ptr, bb.ptr if bias else None, be.at(bc, coff * np.dtype(dt).itemsize),
            {"f32": 0, "f16": 1}[out], M, N, K, mode, lda, ldw, ldc, None)
    if cfg:
        be.tune("gemm_i8_cfg", None)
    flat = be.get(bc, dt, nc)
    got = view(flat, coff, 1, M, N, lc, 0)[0].copy()
    assert np.all(outside(flat, coff, 1, M, N, lc, 0) == dt(SENTINEL)), "wrote outside C"
    acc = a.astype(np.int64) @ w.astype(np.int64).T if M * N * K < 1e8 else np.rint(f64(a) @ f64(w).T)
    part = f64(acc) * f64(sa)[:, None] * f64(sw)
    want = part + (f64(b) if bias and mode != 1 else 0.0)
    tol = 3.01 * U * np.abs(part) + U * np.abs(want)
    if mode:
        want = want + f64(old)
        tol = tol + U * np.abs(want)
    if broken:
        assert np.all(np.isnan(got[M // 2])), "a row with a NaN scale is NaN"
        got[M // 2], want[M // 2], tol[M // 2] = 0, 0, 1
    check(got, want, tol + store_err(want, out) * 1.01 + 1e-44, "product")
    A.unchanged()
    if not mode:
        be.call("mi_gemm_nt_i8", be.at(ba, off), bsa.ptr, be.at(bw, woff), bsw.ptr, bb.ptr if bias else None, be.at(bc, coff * np.dtype(dt).itemsize),
                {"f32": 0, "f16": 1}[out], M, N, K, mode, lda, ldw, ldc, None)
        # by the rules, if the first call was pinned to a build: every build gives the same bits
        assert np.array_equal(be.get(bc, dt, nc).view(np.uint8), flat.view(np.uint8)), "a second call gave other bits"


def broken(be, *, B=2, P, C, G, typ="f32", out="f32", act=1, value="nan", seed=6):
    """A NaN or an infinity in one group of one image leaves NaN in that group, forward and backward (in an 8-bit row's scale), and every
    other group as it is without it."""
    rng = rng_of(seed)
    x = pixels_of(rng, B, P, C, 0.2, 0.0).astype(DT[typ])
    dy = rng.standard_normal((B, P, C)).astype(DT[typ])
    gamma, beta = affine_of(rng, C, "both")
    odt = {"f32": np.float32, "f16": np.float16, "i8": np.int8}[out]
    cg, g, im = C // G, G // 2, B - 1
    hit = np.zeros((B, P, C), bool)
    hit[im, :, g * cg:(g + 1) * cg] = True
    got = []
    for bad in (False, True):
        xx = x.copy()
        if bad:
            xx[im, P // 2, g * cg] = float(value)
        bx, bg, bb, bd = (be.buf(np.ascontiguousarray(t).reshape(-1)) for t in (xx, gamma, beta, dy))
        by, bs = be.buf(np.zeros(B * P * C, odt)), be.buf(np.zeros(B * P, np.float32))
        bo, bdg, bdb = be.buf(np.zeros(B * P * C, DT[typ])), be.buf(np.zeros(C, np.float32)), be.buf(np.zeros(C, np.float32))
        need = be.value("mi_groupnorm_bwd_ws_bytes", B, P, C, G)
        ws = be.buf(np.full(need, 0xff, np.uint8))
        a = MiGroupnormArgs(bx.ptr, bg.ptr, bb.ptr, by.ptr, bs.ptr if out == "i8" else None, None, B, P, C, G, CODE[typ], {"f32": 0, "f16": 1, "i8": I8}[out], act, 1e-5, 0, 0, 0, 0)
        be.call("mi_groupnorm", ctypes.byref(a), ws.ptr, need, None)
        a.y_dtype = CODE[typ]
        q = MiGroupnormBwdArgs(a, bd.ptr, None, bo.ptr, bdg.ptr, bdb.ptr, 0, 0, 0, 0, 0, 0)
        be.call("mi_groupnorm_bwd", ctypes.byref(q), ws.ptr, need, None)
        got.append([f64(be.get(by, odt, B * P * C)).reshape(B, P, C), be.get(bs, np.float32, B * P).reshape(B, P), f64(be.get(bo, DT[typ], B * P * C)).reshape(B, P, C),
                    be.get(bdg, np.float32, C), be.get(bdb, np.float32, C)])
    (y0, s0, d0, g0, b0), (y1, s1, d1, g1, b1) = got
    assert np.array_equal(d1[~hit], d0[~hit]) and np.all(np.isnan(d1[hit]))
    cols = hit[im, 0]
    assert np.array_equal(g1[~cols], g0[~cols]) and np.all(np.isnan(g1[cols])) and np.array_equal(b1[~cols], b0[~cols])
    if out == "i8":
        assert np.array_equal(y1[:im], y0[:im]) and np.array_equal(s1[:im], s0[:im]) and np.all(np.isnan(s1[im])) and np.all(y1[im] == 0)
    else:
        assert np.array_equal(y1[~hit], y0[~hit]) and np.all(np.isnan(y1[hit]))


OPS = {"broken": broken, "groupnorm": groupnorm, "groupnorm_bwd": groupnorm_bwd, "quantize": quantize, "product": product}

# Small shapes where the operators can go wrong, on the emulator and on the GPU.
CASES = {
    "broken": [dict(P=p, C=c, G=g, out=o, value=v, act=a) for p, c, g in ((20, 64, 8), (300, 128, 8), (40, 33, 3), (7, 1024, 512)) for o in ("f32", "i8") for v, a in (("nan", 1), ("inf", 0))]
    + [dict(P=600, C=64, G=2, typ="f16", out="f16", value="-inf")],
    "groupnorm": [
        dict(P=1, C=1, G=1), dict(P=1, C=4, G=4), dict(P=1, C=320, G=32, typ="f16", out="f16", act=1), dict(P=7, C=6, G=2), dict(P=300, C=3, G=1, act=1),
        dict(P=40, C=64, G=8, typ="f16", out="f16", act=1), dict(B=2, P=37, C=320, G=32, act=1), dict(B=3, P=70, C=40, G=4, typ="f16", out="f32"), dict(P=300, C=320, G=32, typ="f16", out="f32", yoff=4), dict(P=1100, C=64, G=2, typ="f16", out="f32", yoff=4, act=1),
        dict(B=2, P=33, C=96, G=32, typ="f32", out="f16", act=1), dict(P=20, C=640, G=32, typ="f16", out="f16"), dict(P=17, C=1000, G=2), dict(P=5, C=2600, G=1),
        dict(P=9, C=1280, G=32, affine="none"), dict(P=9, C=64, G=32, affine="gamma", act=1), dict(P=9, C=64, G=1, affine="beta"),
        # strides, alignment, the images' rows in turn
        dict(B=2, P=19, C=64, G=8, gap=8, ygap=16, typ="f16", out="f16"), dict(B=2, P=19, C=64, G=8, gap=3, ygap=1, act=1), dict(B=3, P=11, C=64, G=8, order="rows", act=1),
        dict(B=3, P=11, C=32, G=8, order="rows", gap=5, typ="f16", out="f16"), dict(P=30, C=64, G=8, off=1), dict(P=30, C=64, G=8, yoff=1), dict(P=30, C=64, G=8, off=4, yoff=8, typ="f16", out="f16"),
        dict(P=30, C=64, G=8, off=8, yoff=8, typ="f16", out="f16"), dict(P=30, C=12, G=3, typ="f16", out="f16"),
        # means far above the spread, outliers where a chunk begins, groups of one value, large and small values, eps 0
        dict(P=200, C=64, G=8, offset=1000.0, act=1), dict(P=200, C=30, G=3, offset=-3e4), dict(P=200, C=64, G=8, outlier=1000.0), dict(P=100, C=30, G=3, outlier=300.0, typ="f16", out="f16"),
        dict(P=50, C=32, G=4, scale=1e15), dict(P=50, C=32, G=4, scale=1e-12, eps=1e-30), dict(P=50, C=32, G=4, eps=0.0), dict(P=50, C=32, G=4, constant=True), dict(P=50, C=33, G=3, constant=True),
        dict(P=64, C=32, G=4, act=1, affine="gamma", offset=0.0, scale=30.0, keep=False), dict(B=40, P=3, C=16, G=4, act=1),
        # several chunks, joined by every workgroup or (many groups) by a launch of their own; some tensors off their 16-byte places
        dict(P=300, C=320, G=32, act=1), dict(B=2, P=301, C=64, G=8, typ="f16", out="f16", offset=300.0), dict(P=700, C=256, G=256, typ="f16", out="f32", act=1), dict(P=300, C=320, G=32, yoff=1), dict(P=300, C=320, G=32, out="i8", yoff=1),
        dict(P=301, C=320, G=32, typ="f16", out="i8"), dict(P=700, C=256, G=256, out="i8", keep=False), dict(P=600, C=37, G=1, outlier=500.0), dict(P=40, C=512, G=512), dict(P=3, C=4096, G=256, typ="f16", out="f16"),
        # a group in a workgroup's registers, at its border and past it; units of two values
        dict(P=256, C=256, G=2, act=1), dict(P=257, C=128, G=1), dict(P=128, C=256, G=1, typ="f16", out="f32"), dict(B=2, P=819, C=20, G=2, typ="f16", out="f16", act=1), dict(P=1639, C=20, G=2),
        dict(P=512, C=64, G=1, act=1), dict(P=513, C=64, G=1), dict(P=1024, C=64, G=1, typ="f16", out="f16", act=1), dict(P=1025, C=64, G=1, typ="f16", out="f16"), dict(P=1300, C=50, G=2, typ="f16", out="f32", offset=200.0), dict(P=16, C=2048, G=2), dict(P=15, C=2052, G=2, act=1), dict(P=100, C=60, G=10, offset=-1000.0, gap=2, ygap=4), dict(P=90, C=64, G=4, off=2, yoff=2, typ="f16", out="f16"),
        # 8-bit rows
        dict(P=1, C=1, G=1, out="i8"), dict(P=20, C=320, G=32, out="i8"), dict(B=2, P=33, C=640, G=32, typ="f16", out="i8"), dict(P=18, C=1280, G=32, typ="f16", out="i8", act=1),
        dict(P=11, C=37, G=1, out="i8", act=1), dict(B=2, P=19, C=64, G=8, ygap=16, gap=4, out="i8"), dict(B=3, P=9, C=64, G=8, order="rows", out="i8", ygap=1),
        dict(P=9, C=2560, G=32, typ="f16", out="i8"), dict(P=9, C=4096, G=32, out="i8"), dict(P=30, C=64, G=8, out="i8", yoff=3), dict(P=50, C=32, G=4, constant=True, affine="none", out="i8"),
    ],
    "groupnorm_bwd": [
        dict(P=1, C=1, G=1), dict(P=1, C=32, G=4, act=1), dict(P=7, C=6, G=2, act=1), dict(P=300, C=3, G=1), dict(P=40, C=64, G=8, typ="f16", dtyp="f16", act=1, res=True),
        dict(B=2, P=37, C=320, G=32, act=1, kept=True), dict(B=3, P=70, C=40, G=4, typ="f16", dtyp="f32"), dict(B=2, P=33, C=96, G=32, dtyp="f16", act=1, res=True),
        dict(P=20, C=640, G=32, typ="f16", dtyp="f16", kept=True), dict(P=17, C=1000, G=2), dict(P=9, C=1280, G=32, affine="none"), dict(P=9, C=64, G=32, affine="gamma", act=1),
        dict(P=9, C=64, G=1, affine="beta", act=1, weights=False), dict(B=2, P=19, C=64, G=8, gap=8, dgap=16, typ="f16", dtyp="f16", res=True),
        dict(B=2, P=19, C=64, G=8, gap=3, dgap=1, act=1, res=True), dict(B=3, P=11, C=64, G=8, order="rows", act=1, kept=True), dict(P=30, C=64, G=8, off=1), dict(P=30, C=64, G=8, doff=1, act=1),
        dict(P=30, C=64, G=8, in_place=True), dict(P=31, C=33, G=3, in_place=True, typ="f16", dtyp="f16", act=1), dict(P=200, C=64, G=8, offset=1000.0), dict(P=200, C=64, G=8, offset=300.0, act=1, kept=True),
        dict(P=50, C=32, G=4, gstd=1e-20), dict(P=50, C=32, G=4, gstd=1e10, act=1), dict(B=40, P=3, C=16, G=4, act=1, res=True), dict(P=5, C=2600, G=1, act=1),
        dict(P=300, C=320, G=32, act=1, res=True), dict(B=2, P=301, C=64, G=8, typ="f16", dtyp="f16", offset=30.0, kept=True), dict(P=700, C=256, G=256, typ="f16", dtyp="f32", act=1), dict(P=300, C=320, G=32, doff=1), dict(P=1100, C=64, G=2, typ="f16", dtyp="f32", off=8, doff=8, act=1), dict(P=1100, C=64, G=2, typ="f16", dtyp="f32", doff=4),
        dict(P=408, C=40, G=1, act=1, res=True), dict(P=409, C=40, G=1, act=1), dict(P=408, C=80, G=2, typ="f16", dtyp="f16", act=1, kept=True), dict(P=409, C=80, G=2, typ="f16", dtyp="f32"), dict(B=3, P=816, C=10, G=1),
        dict(B=2, P=300, C=20, G=2, typ="f16", dtyp="f16", act=1, res=True, gap=2, dgap=2), dict(B=2, P=2, C=2048, G=1, act=1), dict(P=2, C=2052, G=1), dict(P=16, C=2048, G=2, weights=False, kept=True),
        dict(P=400, C=40, G=1, offset=1000.0), dict(B=2, P=520, C=64, G=2, act=1, in_place=True), dict(P=8, C=4096, G=2, typ="f16", dtyp="f32", act=1),
        dict(P=600, C=37, G=1, act=1), dict(P=40, C=512, G=512), dict(P=3, C=4096, G=256, typ="f16", dtyp="f16", weights=False),
    ],
    "quantize": [
        dict(rows=1, cols=1), dict(rows=5, cols=320), dict(rows=9, cols=1280, typ="f16"), dict(rows=6, cols=37), dict(rows=7, cols=37, typ="f16"), dict(rows=3, cols=5120, typ="f16"),
        dict(rows=2, cols=8192), dict(rows=2, cols=8208), dict(rows=4, cols=2048, ldx=2064, ldq=2080), dict(rows=4, cols=64, ldx=67, ldq=65), dict(rows=5, cols=64, off=1, qoff=3),
        dict(rows=5, cols=64, off=2, typ="f16"), dict(rows=12, cols=96, kind="ties"), dict(rows=12, cols=97, kind="ties"), dict(rows=12, cols=96, kind="ties", typ="f16"), dict(rows=12, cols=512, kind="near"),
        dict(rows=12, cols=33, kind="near"), dict(rows=16, cols=64, kind="sizes"), dict(rows=16, cols=65, kind="sizes"), dict(rows=7, cols=64, kind="broken"), dict(rows=7, cols=51, kind="broken", typ="f16"),
        dict(rows=16, cols=64, kind="sizes", typ="f16"),
        # rows that four waves share
        dict(rows=7, cols=784, kind="broken"), dict(rows=7, cols=1552, kind="broken", typ="f16"), dict(rows=12, cols=2048, kind="ties"), dict(rows=4, cols=2816, kind="near", ldx=2832, ldq=2820),
        dict(rows=5, cols=4096, typ="f16"), dict(rows=5, cols=8192, typ="f16", kind="ties"), dict(rows=6, cols=4080, kind="sizes"), dict(rows=3, cols=8192, kind="near"),
    ],
    "product": [
        dict(M=1, N=1, K=1), dict(M=1, N=1, K=16), dict(M=2, N=40, K=64), dict(M=16, N=48, K=320), dict(M=17, N=33, K=48), dict(M=70, N=65, K=144, out="f16"), dict(M=5, N=130, K=37, bias=False),
        dict(M=66, N=70, K=33, out="f16"), dict(M=33, N=64, K=64, mode=1), dict(M=33, N=66, K=80, mode=2), dict(M=33, N=66, K=80, mode=2, out="f16"), dict(M=3, N=70, K=128, mode=2), dict(M=130, N=40, K=256, lda=272, ldw=288, ldc=43),
        dict(M=20, N=40, K=64, lda=65, ldw=67), dict(M=20, N=40, K=64, off=1), dict(M=20, N=40, K=64, woff=8), dict(M=20, N=40, K=64, coff=1, out="f16"), dict(M=20, N=40, K=64, coff=1), dict(M=40, N=40, K=1040, extreme=True), dict(M=4, N=9, K=131071, extreme=True),
        dict(M=9, N=40, K=4096, extreme=True), dict(M=9, N=20, K=64, broken=True), dict(M=40, N=20, K=64, broken=True, mode=2), dict(M=1, N=300, K=1280), dict(M=8, N=20, K=2064, out="f16"), dict(M=77, N=64, K=2048),
        dict(M=150, N=130, K=128, out="f16"), dict(M=300, N=270, K=192), dict(M=260, N=300, K=64, out="f16", ldc=304), dict(M=300, N=260, K=320, mode=2),
        # every build, with tails of rows, columns and codes
        dict(M=20, N=40, K=64, cfg="0"), dict(M=16, N=40, K=80, cfg="1"), dict(M=40, N=40, K=80, cfg="1"), dict(M=1, N=33, K=16, cfg="2"), dict(M=65, N=47, K=2448, cfg="2", extreme=True),
        dict(M=65, N=47, K=2448, cfg="2", out="f16", mode=2), dict(M=1, N=33, K=16, cfg="3"), dict(M=65, N=70, K=400, cfg="3", out="f16"), dict(M=130, N=100, K=272, cfg="3", lda=288, ldw=304, ldc=101),
        dict(M=1, N=33, K=16, cfg="4"), dict(M=129, N=131, K=400, cfg="4", extreme=True), dict(M=140, N=264, K=272, cfg="4", out="f16", mode=2, ldc=272), dict(M=140, N=134, K=128, cfg="4", out="f16"),
        dict(M=1, N=33, K=16, cfg="5"), dict(M=129, N=131, K=400, cfg="5", extreme=True), dict(M=140, N=264, K=656, cfg="5", out="f16", mode=2, ldc=272), dict(M=128, N=128, K=768, cfg="5", out="f16"),
        dict(M=1, N=33, K=16, cfg="6"), dict(M=193, N=259, K=400, cfg="6", extreme=True), dict(M=200, N=264, K=272, cfg="6", out="f16", mode=1), dict(M=1, N=33, K=16, cfg="7"),
        *(dict(M=m + 1, N=n + 1, K=k, cfg=c, extreme=True, **o) for c, m, n in (("3", 64, 64), ("5", 128, 128), ("8", 64, 64)) for k, o in ((16, {}), (128, dict(out="f16")), (400, {}), (528, dict(mode=2, out="f16")), (768, dict(mode=1)))),
        dict(M=257, N=321, K=400, cfg="7", extreme=True), dict(M=260, N=328, K=272, cfg="7", out="f16", mode=2),
    ],
}
# Larger shapes, on the GPU alone: many chunks, tails.
GPU_CASES = {
    "groupnorm": [
        dict(B=2, P=4096, C=640, G=32, typ="f16", out="f16", act=1), dict(P=16385, C=320, G=32, act=1), dict(P=65536, C=128, G=32, typ="f16", out="f16", act=1), dict(B=2, P=1024, C=2560, G=32, typ="f16", out="f16", act=1),
        dict(B=2, P=999, C=1920, G=32, act=1), dict(P=9216, C=960, G=32, typ="f16", out="f32"), dict(P=40000, C=37, G=1, act=1), dict(B=600, P=50, C=64, G=8), dict(B=2, P=2304, C=640, G=32, typ="f16", out="i8"),
        dict(P=1024, C=1280, G=32, out="i8"), dict(P=20000, C=256, G=32, offset=2000.0, act=1), dict(P=20000, C=64, G=8, outlier=5e3), dict(P=3000, C=4096, G=32, typ="f16", out="f16"), dict(P=2000, C=4100, G=4, out="f16"),
        dict(B=2, P=3000, C=512, G=32, gap=64, typ="f16", out="f16", act=1), dict(P=256, C=1280, G=32), dict(P=64, C=1280, G=32, typ="f16", out="f16", act=1), dict(P=257, C=640, G=32, out="i8"),
    ],
    "groupnorm_bwd": [
        dict(B=2, P=4096, C=640, G=32, typ="f16", dtyp="f16", act=1, res=True, kept=True), dict(P=16385, C=320, G=32, act=1), dict(B=2, P=1024, C=2560, G=32, typ="f16", dtyp="f16", act=1),
        dict(P=1024, C=1280, G=32), dict(B=2, P=999, C=1920, G=32, act=1, res=True), dict(P=20000, C=37, G=1, act=1), dict(B=300, P=50, C=64, G=8, act=1), dict(P=3000, C=4096, G=32, typ="f16", dtyp="f16"),
        dict(B=2, P=3000, C=512, G=32, gap=64, dgap=8, typ="f16", dtyp="f16", act=1, res=True), dict(P=256, C=1280, G=32, kept=True),
    ],
    "quantize": [dict(rows=8192, cols=2560, typ="f16"), dict(rows=4099, cols=640), dict(rows=3000, cols=333), dict(rows=2000, cols=1280, kind="near"), dict(rows=777, cols=5120, kind="ties")],
    "product": [
        dict(M=2, N=1280, K=1280), dict(M=1, N=10240, K=1280, out="f16"), dict(M=16, N=5120, K=640), dict(M=77, N=768, K=768), dict(M=154, N=1280, K=2048), dict(M=300, N=1280, K=5120, out="f16"),
        dict(M=2048, N=1280, K=1280, out="f16"), dict(M=1976, N=5120, K=640), dict(M=2100, N=648, K=1312, mode=2), dict(M=4111, N=640, K=2560, out="f16", mode=2), dict(M=333, N=5123, K=320), dict(M=1025, N=2563, K=336, out="f16"),
        dict(M=1000, N=1000, K=999), dict(M=64, N=640, K=5120), dict(M=600, N=640, K=640, lda=656, ldc=1280), dict(M=2048, N=10240, K=1280, out="f16"),
    ],
}
