"""The backward operators against plain 64-bit formulas: cases that run on any backend with the C-ABI (the GPU, or
the CPU emulator of tests/kemu), with error bounds derived from the operators' roundings.

u = 2^-24 is half a step of fp32, h = 2^-11 half a step of fp16, both relative to the value; 2^-25 is half fp16's
smallest step. Sums of n terms in fp32 are bounded by n u sum|terms| along the longest chain of additions.
"""
from __future__ import annotations

import math

import numpy as np

U, H = 2.0 ** -24, 2.0 ** -11
TINY16 = 2.0 ** -25
SENTINEL = 77.0
DT = {"f32": np.float32, "f16": np.float16}
CODE = {"f32": 0, "f16": 1}


def rng_of(seed):
    return np.random.default_rng(seed)


def f64(x):
    return np.asarray(x, dtype=np.float64)


def store_err(x, typ):
    """Half a step of the stored type at |x|."""
    return np.abs(x) * (H if typ == "f16" else U) + (TINY16 if typ == "f16" else 2.0 ** -149)


def check(got, want, tol, what):
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.all(np.isfinite(got)), f"{what}: {np.count_nonzero(~np.isfinite(got))} values are not finite"
    d = np.abs(got - want)
    bad = d > tol
    if np.any(bad):
        i = np.unravel_index(int(np.argmax(d / tol)), d.shape)
        raise AssertionError(f"{what}: {np.count_nonzero(bad)} of {d.size} past their bound; worst at {tuple(map(int, i))}: "
                             f"got {got[i]!r}, want {want[i]!r}, bound {np.broadcast_to(tol, d.shape)[i]:.3e}")
    n = np.linalg.norm(want)
    return float(np.linalg.norm(got - want) / n) if n else 0.0


def rel_check(rel, most, what):
    assert rel <= most, f"{what}: relative error {rel:.3e} > {most:.3e}"


def padded(rng, rows, cols, ld, dtype, std=1.0, off=0):
    """(buffer, view): [rows, cols] normal values at row stride ld, `off` elements into the buffer, gaps of SENTINEL."""
    buf = np.full(off + (rows - 1) * ld + cols if rows else off, SENTINEL, dtype=dtype)
    view = np.lib.stride_tricks.as_strided(buf[off:], (rows, cols), (ld * buf.itemsize, buf.itemsize)) if rows else buf[:0].reshape(0, cols)
    view[...] = (rng.standard_normal((rows, cols)) * std).astype(dtype)
    return buf, view


def strided(flat, off, rows, cols, ld):
    """The [rows, cols] view and a mask of everything else."""
    v = np.lib.stride_tricks.as_strided(flat[off:], (rows, cols), (ld * flat.itemsize, flat.itemsize))
    rest = np.ones(flat.shape, dtype=bool)
    np.lib.stride_tricks.as_strided(rest[off:], (rows, cols), (ld, 1))[...] = False
    return v, rest


class Arena:
    """Buffers of one case: outputs start as SENTINEL, inputs must come back as they were."""

    def __init__(self, be):
        self.be, self.ins = be, []

    def put(self, arr):
        b = self.be.buf(arr)
        self.ins.append((b, arr.copy()))
        return b

    def out(self, n, dtype, init=None):
        return self.be.buf(np.full(n, SENTINEL, dtype=dtype) if init is None else init)

    def unchanged(self):
        for b, a in self.ins:
            got = self.be.get(b, a.dtype, a.size)
            assert np.array_equal(got.view(np.uint8), a.reshape(-1).view(np.uint8)), "an input changed"


# ------------------------------------------------------------------- Q8_0 --

def q8_blocks(w):
    """(34-byte blocks, the float64 values they stand for) of a [rows, cols] weight."""
    b = np.asarray(w, dtype=np.float32).reshape(-1, 32)
    amax = np.abs(b).max(1, keepdims=True)
    d = (amax / 127.0).astype(np.float16)
    q = np.clip(np.rint(b * np.where(amax > 0, 127.0 / np.maximum(amax, 1e-30), 0)), -127, 127).astype(np.int8)
    raw = np.concatenate([d.view(np.uint8).reshape(-1, 2), q.view(np.uint8)], 1).reshape(-1)
    return raw, (q.astype(np.float64) * d.astype(np.float64)).reshape(np.shape(w))


def linear(be, *, typ, M, N, K, mode=0, ldc=0, lda=0, off=0, aoff=0, ws=True, seed=1, std=None, ramp=False, cfg=None, same_as=None):
    """dA = dC . W. `ramp`: dC's rows and columns span many orders of magnitude, with rows of zeros."""
    rng = rng_of(seed)
    dt, ldc_, lda_ = DT[typ], ldc or N, lda or K
    cbuf, dC = padded(rng, M, N, ldc_, dt, std if std is not None else (1e-3 if typ == "f32" else 0.5), off)
    if ramp:
        scale = 10.0 ** rng.uniform(-9, 4, (M, 1)) * 10.0 ** (np.arange(N) * 8.0 / max(N, 1) - 4)
        dC[...] = (dC * scale).astype(dt)
        dC[:: max(1, M // 3)] = 0
    raw, w = q8_blocks(rng.standard_normal((N, K)) * 0.02) if N else (np.zeros(16, np.uint8), np.zeros((0, K)))
    A = Arena(be)
    bC, bW = A.put(cbuf), A.put(raw)
    init = np.full(aoff + (M - 1) * lda_ + K, SENTINEL, dtype=dt)
    if mode:
        strided(init, aoff, M, K, lda_)[0][...] = rng.standard_normal((M, K)).astype(dt)
    old = f64(strided(init, aoff, M, K, lda_)[0]) if mode else 0.0
    bA = A.out(0, dt, init.copy())
    esz = np.dtype(dt).itemsize
    if cfg:
        be.tune("gemm_bwd_cfg", cfg)
    need = be.value("mi_gemm_nt_q8_0_bwd_ws_bytes", M, N, K, CODE[typ]) if ws else 0
    wsb = be.buf(np.full(need, 0xff, np.uint8)) if need else None
    args = (be.at(bC, off * esz), bW.ptr, be.at(bA, aoff * esz), CODE[typ], M, N, K, mode, ldc, lda, wsb.ptr if wsb else None, need, None)
    be.call("mi_gemm_nt_q8_0_bwd", *args)
    flat = be.get(bA, dt, init.size)
    got, rest = strided(flat, aoff, M, K, lda_)
    assert np.all(flat[rest] == SENTINEL), "wrote outside dA"
    x = f64(dC)
    want = x @ w + old
    mag = np.abs(x) @ np.abs(w)
    if typ == "f16":
        # each weight rounded to fp16, fp32 sums, dA rounded
        tol = mag * (H * 1.01 + (N + 8) * U) + np.abs(x).sum(1, keepdims=True) * TINY16 + store_err(want, typ) * 1.01
        most = math.sqrt(2 / 3) * H
    else:
        # pairs: 2^-22 of each operand at most, 2^-22 for the product left out; the pair's absolute floors are 2^-25
        # of weights times 2^6, and of a row whose largest element is at 2^9 or more
        floor = np.abs(x).sum(1, keepdims=True) * 2.0 ** -31 + np.abs(x).max(1, keepdims=True, initial=0) * 2.0 ** -34 * np.abs(w).sum(0)
        tol = mag * (3 * 2.0 ** -22 + (3 * N / 16 + 40) * U) + floor + store_err(want, typ) * 1.01 + 1e-37
        most = 3 * 2.0 ** -22 + math.sqrt(3 * N / 16 + 16) * U
    if mode:
        tol = tol + np.abs(want) * U
    rel = check(got, want, tol, f"linear {typ}")
    if not ramp and N and std is None:
        rel_check(rel, most * (1 if not mode else 1.5), f"linear {typ}")
    A.unchanged()
    first = flat.copy()
    if not mode:  # repeats bit for bit, whatever the workspace held
        be.call("mi_gemm_nt_q8_0_bwd", *args)
        assert np.array_equal(be.get(bA, dt, init.size).view(np.uint8), first.view(np.uint8)), "a second call gave other bits"
    if cfg:
        be.tune("gemm_bwd_cfg", None)


def geglu_parts(v, g, dy):
    cdf = 0.5 * np.vectorize(math.erfc)(-g / math.sqrt(2)) if g.size else g
    pdf = np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return dy * g * cdf, dy * v * (cdf + g * pdf)


def geglu_tol(v, g, dy, dvg, typ):
    """The cdf's approximation is 0.75e-7 off at most; its evaluation (rcp and exp2 to a step, a dozen roundings of values
    under 1, the exponent's three roundings times x^2 / 2 exp(-x^2 / 2) <= 0.37) adds under 6 u: 4.5e-7 in all, and as much
    for x pdf(x); the products three roundings more."""
    e = 4.5e-7
    return (np.abs(dy * g) * e + 4 * U * np.abs(dvg[0]) + store_err(dvg[0], typ) * 1.01,
            np.abs(dy * v) * 2 * e + 4 * U * np.abs(dvg[1]) + store_err(dvg[1], typ) * 1.01)


def geglu_tail_tol(v, g, y, want):
    """Relative bounds where the gates are far below zero. The cdf's tail: the fit 1 u, its coefficients' and the Horner
    form's roundings 10 steps of at most 1.9 times the value (the sum of the coefficients' magnitudes), 3 u of t times
    d ln q / d ln t <= 3, exp2 and two products 6 u, and x^2 u from the exponential's argument and half as much from its
    constant: 35 + 1.5 x^2 in all; x pdf(x) the exponential's alone. Then three products and a sum."""
    cdf = 0.5 * np.vectorize(math.erfc)(-g / math.sqrt(2))
    xpdf = np.abs(g) * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = 1.5 * g * g
    return (np.abs(want[0]) * (38 + k) * U * 1.05 + 1e-37,
            np.abs(y * v) * (cdf * (36 + k) + xpdf * (8 + k)) * U * 1.05 + 3 * U * np.abs(want[1]) + 1e-37)


def geglu(be, *, typ, rows, F, off=0, in_place=False, wide=False, tail=False, seed=2):
    rng = rng_of(seed)
    dt, esz = DT[typ], np.dtype(DT[typ]).itemsize
    h = (rng.standard_normal((rows, 2 * F)) * (6.0 if wide else 1.5)).astype(np.float32)
    dy = (rng.standard_normal((rows, F)) * 0.5).astype(dt)
    if wide and h.size:
        h[0, F:F + min(F, 5)] = [0.0, -0.0, 40.0, -40.0, 1e-30][:min(F, 5)]
    if tail:  # gates from -12 up
        h[:, F:] = np.linspace(-12, 3, rows * F).reshape(rows, F)
    A = Arena(be)
    pad = np.full(off, SENTINEL, dt)
    bdy = A.put(np.concatenate([pad, dy.reshape(-1)]))
    hflat = np.concatenate([np.full(off, SENTINEL, np.float32), h.reshape(-1)])
    if in_place:
        bh = A.out(0, np.float32, hflat)
        bo, hp = bh, be.at(bh, off * 4)
        op = hp
    else:
        bh = A.put(hflat)
        bo = A.out(off + h.size, dt)
        hp, op = be.at(bh, off * 4), be.at(bo, off * esz)
    be.call("mi_geglu_bwd", hp, be.at(bdy, off * esz), op, CODE[typ], rows, F, None)
    flat = be.get(bo, dt, off + h.size)
    assert np.all(flat[:off] == SENTINEL)
    got = flat[off:].reshape(rows, 2 * F)
    v, g, y = f64(h[:, :F]), f64(h[:, F:]), f64(dy)
    want = geglu_parts(v, g, y)
    tol = geglu_tail_tol(v, g, y, want) if tail else geglu_tol(v, g, y, want, typ)
    check(got[:, :F], want[0], tol[0], "geglu dv")
    check(got[:, F:], want[1], tol[1], "geglu dg")
    A.unchanged()


def geglu_gemm(be, *, M, F, K, bias=True, lda=0, lddg=0, lddh=0, off=0, cfg=None, seed=3):
    rng = rng_of(seed)
    lda_, lddg_, lddh_ = lda or K, lddg or F, lddh or 2 * F
    abuf, a = padded(rng, M, K, lda_, np.float16)
    gbuf, dG = padded(rng, M, F, lddg_, np.float16, 0.5, off)
    raw, w = q8_blocks(rng.standard_normal((2 * F, K)) * 0.05)
    b = (rng.standard_normal(2 * F) * 0.05).astype(np.float32)
    A = Arena(be)
    bA, bG, bW, bB = A.put(abuf), A.put(gbuf), A.put(raw), A.put(b)
    n = off + (M - 1) * lddh_ + 2 * F
    bH = A.out(n, np.float16)
    if cfg:
        be.tune("gemm_cfg", cfg)
    be.call("mi_gemm_nt_q8_0_geglu_bwd", bA.ptr, bW.ptr, bB.ptr if bias else None, be.at(bG, 2 * off), be.at(bH, 2 * off), M, F, K,
            lda, lddg, lddh, None)
    if cfg:
        be.tune("gemm_cfg", None)
    flat = be.get(bH, np.float16, n)
    got, rest = strided(flat, off, M, 2 * F, lddh_)
    assert np.all(flat[rest] == SENTINEL), "wrote outside dH"
    x = f64(a)
    hh = x @ w.T + (f64(b) if bias else 0.0)
    eh = (np.abs(x) @ np.abs(w).T) * (H * 1.01 + (K + 8) * U) + np.abs(x).sum(1, keepdims=True) * TINY16 + np.abs(hh) * U
    v, g, y = hh[:, :F], hh[:, F:], f64(dG)
    want = geglu_parts(v, g, y)
    tol = geglu_tol(v, g, y, want, "f16")
    # |gelu'| <= 1.13, |gelu''| <= 0.8
    ev, eg = eh[:, :F], eh[:, F:]
    r0 = check(got[:, :F], want[0], tol[0] + np.abs(y) * 1.13 * eg, "geglu_gemm dv")
    r1 = check(got[:, F:], want[1], tol[1] + np.abs(y) * (1.13 * ev + (np.abs(v) + ev) * 0.8 * eg), "geglu_gemm dg")
    # a rounding is H / sqrt 3 at most in the mean; the weights', entering through v and g, and dH's
    if M * F >= 4096:
        rel_check(max(r0, r1), math.sqrt(3) * H / math.sqrt(3) * 1.2, "geglu_gemm")
    A.unchanged()


# --------------------------------------------------------------- LayerNorm --

def norm(be, *, rows, d, typ="f32", affine=True, res=True, weights=True, in_place=False, off=0, doff=0, offset=0.5, seed=4, eps=1e-5):
    rng = rng_of(seed)
    dt, esz = DT[typ], np.dtype(DT[typ]).itemsize
    x = (rng.standard_normal((rows, d)) * 2 + offset).astype(np.float32)
    dy = (rng.standard_normal((rows, d)) * 0.5).astype(dt)
    gm = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    rs = rng.standard_normal((rows, d)).astype(np.float32)
    A = Arena(be)

    def lead(arr, o):
        return np.concatenate([np.full(o, SENTINEL, arr.dtype), arr.reshape(-1)])

    bx, bdy, bg = A.put(lead(x, off)), A.put(lead(dy, doff)), A.put(gm)
    bo = A.out(0, np.float32, lead(rs, off)) if in_place else A.out(off + x.size, np.float32)
    br = bo if in_place else A.put(lead(rs, off))
    bdg, bdb = A.out(d, np.float32), A.out(d, np.float32)
    need = be.value("mi_layernorm_bwd_ws_bytes", rows, d) if weights else 0
    wsb = be.buf(np.full(max(need, 16), 0xff, np.uint8))
    args = (be.at(bx, off * 4), bg.ptr if affine else None, be.at(bdy, doff * esz), CODE[typ], be.at(br, off * 4) if res else None,
            be.at(bo, off * 4), bdg.ptr if weights else None, bdb.ptr if weights else None, rows, d, eps, wsb.ptr if need else None, need, None)
    be.call("mi_layernorm_bwd", *args)
    X, Y = f64(x), f64(dy)
    mean = X.mean(1, keepdims=True)
    xc = X - mean
    var = (xc * xc).mean(1, keepdims=True)
    inv = 1 / np.sqrt(var + np.float32(eps).astype(np.float64))
    xh = xc * inv
    W = Y * f64(gm) if affine else Y
    c1, c2 = W.mean(1, keepdims=True), (W * xh).mean(1, keepdims=True)
    want = inv * (W - c1 - xh * c2) + (f64(rs) if res else 0.0)
    # chains: d / 64 additions a lane and six across the wave, then a division
    n = d / 64 + 4 + 8
    e_mean = n * U * np.abs(X).mean(1, keepdims=True)
    e_xc = e_mean + U * (np.abs(X) + np.abs(mean))
    # the variance about a mean that is off: its square; then the sum, the square root and the reciprocal
    e_inv = inv * ((n + 8) * U + inv * inv * (e_mean ** 2 + 2 * np.sqrt(var) * U * np.abs(X).max(1, keepdims=True, initial=0)))
    e_xh = inv * e_xc + np.abs(xc) * e_inv + 2 * U * np.abs(xh)
    e_w = U * np.abs(W)
    e_c1 = (n * U) * np.abs(W).mean(1, keepdims=True) + e_w.mean(1, keepdims=True)
    e_c2 = (n * U) * np.abs(W * xh).mean(1, keepdims=True) + (np.abs(W) * e_xh + e_w * np.abs(xh)).mean(1, keepdims=True)
    body = np.abs(W) + np.abs(c1) + np.abs(xh * c2)
    tol = e_inv * body + inv * (e_w + e_c1 + np.abs(xh) * e_c2 + e_xh * np.abs(c2) + 4 * U * body) + 2 * U * (np.abs(want) + (np.abs(rs) if res else 0))
    flat = be.get(bo, np.float32, off + x.size)
    assert np.all(flat[:off] == SENTINEL)
    check(flat[off:].reshape(rows, d), want, tol + 1e-37, "norm dx")
    dg, db = be.get(bdg, np.float32, d), be.get(bdb, np.float32, d)
    if weights:
        chain = 64 + rows / 1024 + 32
        tg = (np.abs(Y) * e_xh).sum(0) + chain * U * np.abs(Y * xh).sum(0) + 1e-37
        check(dg, (Y * xh).sum(0), tg, "norm dgamma")
        check(db, Y.sum(0), chain * U * np.abs(Y).sum(0) + 1e-37, "norm dbeta")
    else:
        assert np.all(dg == np.float32(SENTINEL)) and np.all(db == np.float32(SENTINEL))
    A.unchanged()
    if not in_place:
        be.call("mi_layernorm_bwd", *args)
        assert np.array_equal(be.get(bo, np.float32, off + x.size).view(np.uint8), flat.view(np.uint8))
        assert np.array_equal(be.get(bdg, np.float32, d).view(np.uint8), dg.view(np.uint8))
        assert np.array_equal(be.get(bdb, np.float32, d).view(np.uint8), db.view(np.uint8))


# --------------------------------------------------------------- attention --

def softmax_rows(S):
    top = S.max(-1, keepdims=True, initial=-np.inf)
    E = np.exp(S - np.where(np.isfinite(top), top, 0.0))
    t = E.sum(-1, keepdims=True)
    return E / np.where(t > 0, t, 1.0)


def attn_head(q, k, v, do, scale, seen, typ, o_stored):
    """One head in 64 bits: (dq, dk, dv), and bounds of what the kernels' roundings do to them.

    o_stored: the output as the caller has it, rounded to its type: delta comes from it."""
    S = np.where(seen, (q @ k.T) * scale, -np.inf)
    P = softmax_rows(S)
    dP = do @ v.T
    delta = (do * o_stored).sum(1, keepdims=True)
    true_delta = (P * dP).sum(1, keepdims=True)
    dS = P * (dP - true_delta)
    want = (scale * dS @ k, scale * dS.T @ q, P.T @ do)
    T = max(q.shape[0], k.shape[0])
    f16 = typ == "f16"
    aq, ak, av, ag = np.abs(q), np.abs(k), np.abs(v), np.abs(do)
    gm, gr = ag.max(initial=0.0), ag.max(1, keepdims=True, initial=0.0)
    # a pair leaves 2^-22 of each operand and of the product of the low parts, and not less than 2^-25 of an operand as it
    # is held: q, k and v as they are, dO with its largest element at 2^8 or more (of the row, or of the head)
    pair, low = (0.0, 0.0) if f16 else (3 * 2.0 ** -22, TINY16)
    gq, gk = (0.0, 0.0) if f16 else (gr * 2.0 ** -33, gm * 2.0 ** -33)
    # scores: 64 terms; the exponent's fma, its argument, the row's maximum and log2 sum in fp32, at the size of the
    # largest score seen; exp2 and the sum
    eS = abs(scale) * ((aq @ ak.T) * (pair + 16 * U) + low * (aq.sum(1, keepdims=True) + ak.sum(1)[None, :]))
    top = np.where(np.isfinite(S), np.abs(S), 0.0).max(1, keepdims=True, initial=0.0) + np.log(T + 1)
    eP = P * (eS + eS.max(1, keepdims=True, initial=0.0) + 12 * U * top + (16 + T / 16) * U) * 1.1
    ed = np.abs(delta - true_delta) + (ag * np.abs(o_stored)).sum(1, keepdims=True) * 70 * U
    adP = ag @ av.T
    # P and dS as operands: fp16 rounds them (H), a pair leaves 2^-22; not less than 2^-25 of what they are held at:
    # P 2^14; dS in the key kernel 2^14 over the head's bound of |dP - delta|, to within a factor of two; in the query
    # kernel exp2(s - m) (l is 1 at least) with the row's largest |dO| at 2^-4 (fp16) or 2^2 (fp32), or, where the row's dS
    # would pass 2^15 there, with its largest (|dP - delta| at most) at 2^13 or more
    r = H * 1.01 if f16 else 2.0 ** -22
    fP = TINY16 * 2.0 ** -14
    fK = TINY16 * 2.0 ** -13 * (64 * gm * av.max(initial=0.0) + np.abs(delta).max(initial=0.0))
    fQ = TINY16 * (gr * (2.0 ** 4 if f16 else 2.0 ** -2) + 2.0 ** -13 * np.abs(dP - true_delta).max(1, keepdims=True, initial=0.0))
    chain = (T + 64) * U + pair

    def d_score(gfloor, floor):
        edP = adP * (pair + 16 * U) + gfloor * av.sum(1)[None, :] + low * ag.sum(1, keepdims=True)
        e = P * (edP + ed) + eP * (np.abs(dP) + np.abs(true_delta) + edP + ed) + 6 * U * np.abs(dS)
        return e + (np.abs(dS) + e) * r + floor * seen

    eq, ek = d_score(gq, fQ), d_score(gk, fK)
    aD = np.abs(dS)
    e_dq = abs(scale) * (eq @ (ak + low) + aD @ (chain * ak + low))
    e_dk = abs(scale) * (ek.T @ (aq + low) + aD.T @ (chain * aq + low))
    e_p = eP + (P + eP) * r + fP * seen
    e_dv = e_p.T @ (ag + gk) + P.T @ (chain * ag + gk)
    return want, (e_dq, e_dk, e_dv)


def attention(be, *, typ, batch=1, Tq, Tk, heads=1, hd=64, causal=False, lens=None, scale=0.0, gap=0, off=0, joint=False, gstd=None,
              grow=False, peak=1.0, vsize=0.0, vblocks=(), seed=5, poison=False, norm_check=True):
    rng = rng_of(seed)
    dt, esz, C = DT[typ], np.dtype(DT[typ]).itemsize, heads * hd
    ld = 3 * C if joint else C + gap
    std = gstd if gstd is not None else (1e-3 if typ == "f32" else 0.5)

    def tensor(T, sd=1.0):
        x = (rng.standard_normal((batch, T, C)) * sd).astype(dt)
        return x

    q, k, v, do = tensor(Tq, peak), tensor(Tk), tensor(Tk), tensor(Tq, std)
    if vsize:  # values of this size, each key's of one sign, and the gradients of one: no product cancels another
        v = (np.sign(rng.standard_normal((batch, Tk, 1))) * np.abs(f64(v)) * vsize).astype(dt)
        do = np.abs(do)
    for k0, k1, factor in vblocks:  # values of these keys times factor
        v[:, k0:k1] = (f64(v[:, k0:k1]) * factor).astype(dt)
    if grow:  # queries' gradients from 1e-6 to 1e2 of std, some zero
        do = (f64(do) * 10.0 ** rng.uniform(-3 if typ == "f16" else -6, 2, (batch, Tq, 1))).astype(dt)
        do[:, ::7] = 0
    sc = scale if scale else 1 / math.sqrt(hd)
    L = [Tk] * batch if lens is None else [min(max(x, 0), Tk) for x in lens]
    i, j = np.arange(Tq)[:, None], np.arange(Tk)[None, :]
    seen = [(j < L[b]) & ((j <= i) if causal else True) & (i >= 0) for b in range(batch)]
    out = np.zeros((batch, Tq, C))
    for b in range(batch):
        for h in range(heads):
            c = slice(h * hd, (h + 1) * hd)
            S = np.where(seen[b], f64(q[b, :, c]) @ f64(k[b, :, c]).T * sc, -np.inf)
            out[b, :, c] = softmax_rows(S) @ f64(v[b, :, c])
    o = out.astype(dt)
    if poison and lens is not None:  # what lies behind a row's keys is not read
        for b in range(batch):
            k[b, L[b]:], v[b, L[b]:] = np.nan, np.inf

    A = Arena(be)

    def place(x, l=ld):
        T = x.shape[1]
        buf = np.full(off + batch * T * l, SENTINEL, dtype=dt)
        if x.size:
            np.lib.stride_tricks.as_strided(buf[off:], x.shape, (T * l * esz, l * esz, esz))[...] = x
        return buf

    keep = [A.put(place(x)) for x in (q, k, v, o, do)]
    pq, pk, pv, po, pg = (be.at(x, off * esz) for x in keep)
    if joint:
        n = off + batch * max(Tq, Tk) * ld
        g = A.out(n, dt)
        bufs = [(g, n, i * C) for i in range(3)]
    else:
        sizes = [off + batch * T * ld for T in (Tq, Tk, Tk)]
        bufs = [(A.out(n, dt), n, 0) for n in sizes]
    pd = [be.at(b, (off + o_) * esz) for b, _, o_ in bufs]
    bl = A.put(np.asarray(lens, np.int32)) if lens is not None else None

    import ctypes

    from sdvk_amd._lib import MiAttnArgs, MiAttnBwdArgs
    f = MiAttnArgs(q=pq, k=pk, v=pv, out=po, batch=batch, Tq=Tq, Tk=Tk, C=C, heads=heads, causal=int(causal), in_dtype=CODE[typ],
                   out_dtype=CODE[typ], ldq=ld, ldk=ld, ldv=ld, ldo=ld, kv_len=bl.ptr if bl else None, scale=scale)
    x = MiAttnBwdArgs(fwd=f, dout=pg, dq=pd[0], dk=pd[1], dv=pd[2], lddout=ld, lddq=ld, lddk=ld, lddv=ld)
    need = be.value("mi_fused_attention_bwd_ws_bytes", ctypes.byref(x))
    wsb = be.buf(np.full(max(need, 16), 0xff, np.uint8))
    args = (ctypes.byref(x), wsb.ptr, need, None)
    be.call("mi_fused_attention_bwd", *args)

    flats = [be.get(b, dt, n) for b, n, _ in bufs]
    grads = []
    rests = [np.ones(fl.shape, bool) for fl in flats]
    for (b, n, o_), fl, T, rest in zip(bufs, flats, (Tq, Tk, Tk), rests):
        st = (T * ld, ld, 1)
        grads.append(np.lib.stride_tricks.as_strided(fl[off + o_:], (batch, T, C), tuple(s * esz for s in st)))
        np.lib.stride_tricks.as_strided(rest[off + o_:], (batch, T, C), st)[...] = False
    if joint:
        rests = [rests[0] & rests[1] & rests[2]] * 3
    for fl, rest in zip(flats, rests):
        assert np.all(fl[rest] == SENTINEL), "wrote outside the gradients"
    rels = [[], [], []]
    kz, vz = (np.where(np.isfinite(f64(t)), f64(t), 0.0) for t in (k, v))
    for b in range(batch):
        for h in range(heads):
            c = slice(h * hd, (h + 1) * hd)
            want, tol = attn_head(f64(q[b, :, c]), kz[b, :, c], vz[b, :, c], f64(do[b, :, c]), sc, seen[b], typ, f64(o[b, :, c]))
            for n, (got, w, t) in enumerate(zip(grads, want, tol)):
                rels[n].append(check(got[b, :, c], w, t * 1.02 + store_err(w, typ) * 1.01 + 1e-37, f"attention d{'qkv'[n]} batch {b} head {h}"))
            for n in (1, 2):
                assert np.all(grads[n][b, L[b]:, c] == 0), "a key past its row's length has a gradient"
    if norm_check and Tq * Tk >= 4096 and not grow and scale == 0 and peak == 1:
        # independent roundings, H / sqrt 3 each at most: P or dS, the result, and delta's (from the stored output) where a
        # row has few keys (a peaked row's dS is the small difference of dP and delta: the bounds above hold it). fp32:
        # 2^-22 of the operands of three products and of what is left out of them, 8 units of it in all
        most = H if typ == "f16" else 8 * 2.0 ** -22
        for n in range(3):
            rel_check(max(rels[n]), most, f"attention d{'qkv'[n]}")
    A.unchanged()
    be.call("mi_fused_attention_bwd", *args)
    for (b, n, _), fl in zip(bufs, flats):
        assert np.array_equal(be.get(b, dt, n).view(np.uint8), fl.view(np.uint8)), "a second call gave other bits"


OPS = {"attention": attention, "linear": linear, "geglu": geglu, "geglu_gemm": geglu_gemm, "norm": norm}

# Small shapes where the operators can go wrong, on the emulator and on the GPU.
CASES = {
    "attention": [
        dict(typ="f16", Tq=1, Tk=1), dict(typ="f32", Tq=1, Tk=1), dict(typ="f16", Tq=1, Tk=100, heads=2), dict(typ="f32", Tq=100, Tk=1, heads=2),
        dict(typ="f16", Tq=100, Tk=150, heads=2), dict(typ="f32", Tq=70, Tk=130, heads=2), dict(typ="f16", Tq=130, Tk=77, batch=2, heads=2, lens=[77, 13]),
        dict(typ="f32", Tq=66, Tk=77, batch=2, lens=[64, 1]), dict(typ="f16", Tq=65, Tk=70, batch=3, lens=[0, 65, -2], poison=True),
        dict(typ="f32", Tq=33, Tk=70, batch=3, lens=[0, 64, 700], poison=True), dict(typ="f16", Tq=140, Tk=140, causal=True, heads=2),
        dict(typ="f32", Tq=140, Tk=140, causal=True), dict(typ="f16", Tq=70, Tk=200, causal=True), dict(typ="f32", Tq=200, Tk=70, causal=True),
        dict(typ="f16", Tq=77, Tk=77, causal=True, batch=2, lens=[77, 5]),
        dict(typ="f16", Tq=70, Tk=200, causal=True, heads=3), dict(typ="f32", Tq=100, Tk=300, causal=True, batch=2),
        # head widths, rows off their 16-byte places, gaps, the joint [rows, 3C] gradient
        dict(typ="f16", Tq=70, Tk=66, heads=3, hd=40), dict(typ="f32", Tq=70, Tk=66, heads=3, hd=40), dict(typ="f16", Tq=40, Tk=70, heads=2, hd=20),
        dict(typ="f32", Tq=40, Tk=70, heads=2, hd=20), dict(typ="f16", Tq=40, Tk=70, heads=2, hd=37), dict(typ="f32", Tq=40, Tk=70, heads=3, hd=1),
        dict(typ="f16", Tq=40, Tk=70, heads=2, off=1), dict(typ="f32", Tq=40, Tk=70, heads=2, off=1, gap=3), dict(typ="f16", Tq=40, Tk=70, heads=2, gap=8, off=8),
        dict(typ="f16", Tq=70, Tk=70, heads=2, joint=True), dict(typ="f32", Tq=70, Tk=70, heads=2, joint=True, batch=2),
        # scales, peaked rows, gradients of many sizes
        dict(typ="f16", Tq=40, Tk=70, scale=-0.2), dict(typ="f32", Tq=40, Tk=70, scale=-0.2), dict(typ="f16", Tq=40, Tk=140, peak=30.0),
        dict(typ="f32", Tq=40, Tk=140, peak=30.0), dict(typ="f16", Tq=140, Tk=70, grow=True), dict(typ="f32", Tq=140, Tk=70, grow=True),
        dict(typ="f32", Tq=40, Tk=70, gstd=1e-20), dict(typ="f32", Tq=40, Tk=70, gstd=1e10), dict(typ="f16", Tq=40, Tk=70, gstd=2.0 ** -20, norm_check=False),
        dict(typ="f16", Tq=70, Tk=150, vsize=2000.0, gstd=0.01, norm_check=False), dict(typ="f32", Tq=70, Tk=150, vsize=2000.0, norm_check=False),
        dict(typ="f16", Tq=40, Tk=70, vsize=100.0, causal=True, peak=5.0, gstd=0.1, norm_check=False),
        dict(typ="f16", Tq=40, Tk=70, gstd=0.0), dict(typ="f32", Tq=0, Tk=5), dict(typ="f16", Tq=5, Tk=0),
        # blocks of 128 keys whose values are all zero, next to others: whole, one key, packed, causal, shared by workgroups
        *(dict(typ=t, norm_check=False, **c) for t in ("f16", "f32") for c in (
            dict(Tq=40, Tk=150, vblocks=[[128, 150, 0.0]]), dict(Tq=64, Tk=129, vblocks=[[128, 129, 0.0]]),
            dict(Tq=40, Tk=154, hd=40, off=1, vblocks=[[77, 154, 0.0]]), dict(Tq=128, Tk=256, gstd=100.0, vblocks=[[128, 256, 0.0]]),
            dict(Tq=200, Tk=200, causal=True, heads=2, vblocks=[[128, 200, 0.0]]), dict(Tq=600, Tk=150, heads=2, vblocks=[[128, 150, 0.0]]),
            dict(Tq=40, Tk=300, batch=2, lens=[300, 129], gstd=100.0, vblocks=[[100, 256, 0.0]], poison=True),
            dict(Tq=40, Tk=70, vblocks=[[0, 70, 0.0]]))),
        dict(typ="f32", Tq=40, Tk=70, gstd=1e12, vblocks=[[0, 70, 0.0]], norm_check=False), dict(typ="f32", Tq=40, Tk=150, gstd=1e12, vblocks=[[128, 150, 0.0]], norm_check=False),
        dict(typ="f32", Tq=40, Tk=70, gstd=2e29, vblocks=[[0, 35, 1e3]], norm_check=False), dict(typ="f32", Tq=40, Tk=70, gstd=1e-30),
        # large gradients on small values, so that the weights' and the scores' powers of two lie far apart
        dict(typ="f16", Tq=40, Tk=400, gstd=3000.0, peak=6.0, norm_check=False), dict(typ="f16", Tq=128, Tk=256, gstd=8000.0, vblocks=[[128, 256, 2.0 ** -24]], norm_check=False),
        dict(typ="f16", Tq=128, Tk=256, gstd=8000.0, vblocks=[[128, 256, 2.0 ** -20]], norm_check=False), dict(typ="f16", Tq=128, Tk=256, gstd=100.0, vblocks=[[128, 256, 1e-7]], norm_check=False),
        dict(typ="f16", Tq=40, Tk=400, gstd=3000.0, peak=6.0, hd=40, off=1, norm_check=False), dict(typ="f16", Tq=140, Tk=140, gstd=3000.0, peak=4.0, causal=True, norm_check=False),
        dict(typ="f16", Tq=64, Tk=70, gstd=0.5, vblocks=[[0, 70, 2.0 ** -24]], norm_check=False), dict(typ="f16", Tq=64, Tk=200, gstd=1e-6, vblocks=[[0, 128, 2.0 ** -23], [128, 200, 1e4]], norm_check=False),
        # parts of the queries
        dict(typ="f16", batch=541, Tq=3, Tk=5, hd=8), dict(typ="f16", Tq=300, Tk=40, heads=2), dict(typ="f32", Tq=260, Tk=140), dict(typ="f16", Tq=300, Tk=140, causal=True),
    ],
    "linear": [
        dict(typ="f16", M=1, N=1, K=32), dict(typ="f32", M=1, N=1, K=32), dict(typ="f16", M=3, N=8, K=96),
        dict(typ="f32", M=2, N=96, K=64), dict(typ="f16", M=130, N=72, K=160), dict(typ="f32", M=70, N=36, K=160),
        # N that takes element-wise loads, rows of dC and dA off their 16-byte places, gaps between rows
        dict(typ="f16", M=67, N=37, K=64), dict(typ="f32", M=66, N=37, K=96), dict(typ="f16", M=65, N=64, K=64, off=3, aoff=1),
        dict(typ="f32", M=65, N=64, K=64, off=1, aoff=3, lda=67), dict(typ="f16", M=33, N=64, K=64, ldc=72, lda=72),
        dict(typ="f32", M=33, N=64, K=64, ldc=68, lda=68, mode=1), dict(typ="f16", M=33, N=64, K=64, ldc=67, lda=65, mode=1),
        # parts of N with and without a workspace
        dict(typ="f16", M=40, N=640, K=96, mode=1), dict(typ="f32", M=40, N=640, K=96), dict(typ="f32", M=40, N=640, K=96, ws=False),
        # rows of many sizes; sizes that grow along a row, so that the exponents fall again and again
        dict(typ="f32", M=37, N=320, K=64, ramp=True), dict(typ="f32", M=20, N=320, K=64, ramp=True, ws=False),
        dict(typ="f32", M=9, N=64, K=32, std=1e-30), dict(typ="f32", M=9, N=64, K=32, std=1e25),
        dict(typ="f16", M=5, N=0, K=64), dict(typ="f32", M=5, N=0, K=64, mode=1),
        # few rows: every number of them that has a kernel, N past one pass of the workgroup
        dict(typ="f16", M=1, N=2100, K=32), dict(typ="f32", M=2, N=1025, K=64, ramp=True), dict(typ="f32", M=4, N=1030, K=32, mode=1),
        dict(typ="f16", M=3, N=530, K=96, off=3, aoff=1, ldc=533, lda=97), dict(typ="f32", M=4, N=513, K=64, off=1, aoff=1, lda=65),
        dict(typ="f32", M=3, N=64, K=32, std=1e-30), dict(typ="f16", M=3, N=40, K=64, cfg="2:1"),
        # every tile build, alone and with parts
        dict(typ="f16", M=300, N=136, K=288, cfg="0"), dict(typ="f32", M=300, N=68, K=288, cfg="0", mode=1),
        dict(typ="f16", M=150, N=200, K=288, cfg="1:3"), dict(typ="f32", M=150, N=100, K=160, cfg="1:2"),
        dict(typ="f16", M=150, N=200, K=160, cfg="2:2"), dict(typ="f32", M=70, N=100, K=96, cfg="2:3", mode=1),
        dict(typ="f16", M=260, N=64, K=160, cfg="0", lda=161), dict(typ="f32", M=130, N=96, K=160, cfg="1", ws=False),
        dict(typ="f32", M=300, N=100, K=288, cfg="3:2"), dict(typ="f32", M=260, N=100, K=320, cfg="3", mode=1), dict(typ="f32", M=200, N=320, K=96, cfg="3", ramp=True),
        dict(typ="f32", M=260, N=320, K=160, cfg="0", ramp=True), dict(typ="f32", M=130, N=320, K=160, cfg="1", ramp=True),
    ],
    "geglu": [
        dict(typ="f32", rows=3, F=64), dict(typ="f16", rows=5, F=36), dict(typ="f32", rows=7, F=37), dict(typ="f16", rows=4, F=1),
        dict(typ="f32", rows=2, F=64, off=1), dict(typ="f16", rows=3, F=64, off=1), dict(typ="f32", rows=5, F=40, in_place=True),
        dict(typ="f32", rows=40, F=100, tail=True), dict(typ="f32", rows=40, F=101, tail=True),
        dict(typ="f32", rows=5, F=41, in_place=True), dict(typ="f32", rows=40, F=100, wide=True), dict(typ="f16", rows=40, F=100, wide=True),
    ],
    "geglu_gemm": [
        dict(M=1, F=1, K=32), dict(M=2, F=24, K=64), dict(M=16, F=40, K=160), dict(M=5, F=37, K=64, bias=False),
        dict(M=77, F=48, K=64), dict(M=130, F=100, K=96), dict(M=70, F=37, K=128, lddg=41, lddh=80), dict(M=65, F=40, K=64, off=2),
        dict(M=33, F=64, K=128, lda=136, lddg=72, lddh=136), dict(M=300, F=130, K=256, cfg="0"), dict(M=200, F=130, K=128, cfg="5"),
        dict(M=140, F=130, K=128, cfg="6", bias=False), dict(M=70, F=40, K=128, cfg="1"), dict(M=70, F=100, K=192, cfg="2"),
        dict(M=70, F=40, K=128, cfg="3"), dict(M=260, F=70, K=128, cfg="4"),
    ],
    "norm": [
        dict(rows=1, d=4), dict(rows=1, d=1), dict(rows=9, d=1280), dict(rows=5, d=640, typ="f16"), dict(rows=7, d=37), dict(rows=6, d=37, typ="f16"),
        dict(rows=3, d=4096), dict(rows=3, d=4100), dict(rows=4, d=2000, res=False), dict(rows=4, d=320, affine=False), dict(rows=4, d=320, weights=False),
        dict(rows=5, d=64, in_place=True), dict(rows=5, d=65, in_place=True, typ="f16"), dict(rows=5, d=64, off=1), dict(rows=5, d=64, doff=1, typ="f16"),
        dict(rows=130, d=68), dict(rows=150, d=33), dict(rows=6, d=256, offset=300.0), dict(rows=6, d=255, offset=-300.0), dict(rows=4, d=512, weights=False, affine=False, res=False),
    ],
}
# Larger shapes, on the GPU alone: grids that stride over rows, splits as the rules choose them, tails.
GPU_CASES = {
    "attention": [
        # more than 512 blocks of few tiles, not a multiple of the workgroups
        dict(typ="f32", batch=7, heads=11, Tq=800, Tk=77, hd=8), dict(typ="f16", batch=7, heads=11, Tq=800, Tk=40, hd=8),
        dict(typ="f16", batch=11, heads=7, Tq=77, Tk=1000, hd=16, causal=True),
        # more than 512 blocks, some whole and the others shared
        dict(typ="f32", heads=77, Tq=900, Tk=1200, hd=4),
        dict(typ="f16", Tq=1024, Tk=1024, heads=4, batch=2), dict(typ="f16", Tq=1024, Tk=77, heads=20, batch=2, lens=[77, 30]),
        dict(typ="f32", Tq=900, Tk=900, heads=4), dict(typ="f32", Tq=1000, Tk=154, heads=5, batch=2, lens=[154, 100]), dict(typ="f16", Tq=2000, Tk=2000, heads=2),
        dict(typ="f16", Tq=1500, Tk=1500, heads=2, causal=True), dict(typ="f32", Tq=1100, Tk=1100, heads=2, causal=True), dict(typ="f32", Tq=77, Tk=77, heads=12, causal=True),
        dict(typ="f16", Tq=17, Tk=3000, heads=3), dict(typ="f32", Tq=5, Tk=2000, heads=2, hd=40), dict(typ="f16", Tq=3000, Tk=17, heads=3),
        dict(typ="f16", Tq=1000, Tk=1000, heads=3, hd=20), dict(typ="f32", Tq=600, Tk=700, heads=3, hd=40),
    ],
    "linear": [
        dict(typ="f32", M=2, N=1280, K=1280), dict(typ="f16", M=16, N=1280, K=640), dict(typ="f16", M=77, N=640, K=2048),
        dict(typ="f32", M=154, N=1280, K=2048), dict(typ="f16", M=1000, N=640, K=2560), dict(typ="f32", M=577, N=1280, K=1280),
        dict(typ="f16", M=2100, N=648, K=1312), dict(typ="f32", M=2100, N=640, K=1312, mode=1), dict(typ="f32", M=513, N=1000, K=640, ramp=True),
        dict(typ="f16", M=4111, N=130, K=640, lda=648), dict(typ="f16", M=333, N=5120, K=320),
    ],
    "geglu": [dict(typ="f32", rows=2050, F=1280), dict(typ="f16", rows=1111, F=1276), dict(typ="f32", rows=700, F=1277)],
    "geglu_gemm": [dict(M=1025, F=640, K=320), dict(M=2048, F=1280, K=640), dict(M=3, F=2560, K=640), dict(M=700, F=1277, K=640, bias=False)],
    "norm": [dict(rows=2100, d=1280), dict(rows=4099, d=640, typ="f16"), dict(rows=3000, d=333), dict(rows=70000, d=8), dict(rows=1, d=768, typ="f16")],
}
