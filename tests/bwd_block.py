"""The backward operators run together: the gradients of a transformer block (self attention, attention to a context,
GEGLU feed-forward, each behind a LayerNorm and a residual) with frozen Q8_0 weights, through sdvk_amd.ops, against the same
in 64 bits and against differences of the 64-bit forward pass.

Runs on any backend with buffers (bwd_ref): the GPU, or the CPU emulator.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

import bwd_ref
from bwd_ref import H, U, f64, q8_blocks, rng_of, softmax_rows

EPS = 1e-5
SIZES = dict(batch=2, T=70, C=128, heads=2, F=160, Tc=77, Cc=96, lens=(77, 40))
INNER = ("dG", "dh", "dn3", "dx2", "do2", "dq2", "dk2", "dv2", "dn2", "dx1", "do1", "dqkv", "dn1")
RESULTS = ("dx", "dctx", "dg1", "db1", "dg2", "db2", "dg3", "db3")


def norm_fwd(x, gm, bt):
    xc = x - x.mean(-1, keepdims=True)
    return xc / np.sqrt((xc * xc).mean(-1, keepdims=True) + EPS) * gm + bt


def norm_bwd(x, gm, dy):
    xc = x - x.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((xc * xc).mean(-1, keepdims=True) + EPS)
    xh, w = xc * inv, dy * gm
    dx = inv * (w - w.mean(-1, keepdims=True) - xh * (w * xh).mean(-1, keepdims=True))
    return dx, (dy * xh).reshape(-1, x.shape[-1]).sum(0), dy.reshape(-1, x.shape[-1]).sum(0)


def gelu(g):
    return g * 0.5 * np.vectorize(math.erfc)(-g / math.sqrt(2))


class Block:
    """Weights, inputs and the 64-bit passes."""

    def __init__(self, seed=11, batch=2, T=70, C=128, heads=2, F=160, Tc=77, Cc=96, lens=(77, 40)):
        r = rng_of(seed)
        self.__dict__.update(batch=batch, T=T, C=C, heads=heads, F=F, Tc=Tc, Cc=Cc, lens=lens)
        shapes = dict(wqkv=(3 * C, C), wo=(C, C), wq2=(C, C), wk2=(C, Cc), wv2=(C, Cc), wo2=(C, C), w1=(2 * F, C), w2=(C, F))
        self.raw, self.w = {}, {}
        for n, s in shapes.items():
            self.raw[n], self.w[n] = q8_blocks(r.standard_normal(s) / math.sqrt(s[1]))
        self.v = {}
        for i in (1, 2, 3):
            self.v[f"g{i}"] = (1 + 0.2 * r.standard_normal(C)).astype(np.float32)
            self.v[f"b{i}"] = (0.2 * r.standard_normal(C)).astype(np.float32)
        self.v["bias1"] = (0.1 * r.standard_normal(2 * F)).astype(np.float32)
        self.x = r.standard_normal((batch, T, C)).astype(np.float32)
        self.ctx = r.standard_normal((batch, Tc, Cc)).astype(np.float32)
        self.dy = (1e-3 * r.standard_normal((batch, T, C))).astype(np.float32)

    def heads_of(self, t):
        return t.reshape(t.shape[0], t.shape[1], self.heads, -1).transpose(0, 2, 1, 3)

    def seen(self, cross):
        if not cross:
            return np.ones((self.batch, 1, 1, self.T), bool)
        return (np.arange(self.Tc)[None, :] < np.asarray(self.lens)[:, None])[:, None, None, :]

    def attn(self, q, k, v, cross):
        q, k, v = map(self.heads_of, (q, k, v))
        S = np.where(self.seen(cross), q @ k.transpose(0, 1, 3, 2) / math.sqrt(q.shape[-1]), -np.inf)
        o = softmax_rows(S) @ v
        return o.transpose(0, 2, 1, 3).reshape(o.shape[0], o.shape[2], -1)

    def attn_bwd(self, q, k, v, do, cross):
        q, k, v, do = map(self.heads_of, (q, k, v, do))
        sc = 1 / math.sqrt(q.shape[-1])
        P = softmax_rows(np.where(self.seen(cross), q @ k.transpose(0, 1, 3, 2) * sc, -np.inf))
        dP = do @ v.transpose(0, 1, 3, 2)
        dS = P * (dP - (P * dP).sum(-1, keepdims=True))
        back = lambda t: t.transpose(0, 2, 1, 3).reshape(t.shape[0], t.shape[2], -1)  # noqa: E731
        return back(sc * dS @ k), back(sc * dS.transpose(0, 1, 3, 2) @ q), back(P.transpose(0, 1, 3, 2) @ do)

    def forward(self, x, ctx):
        w, v, C = self.w, {n: f64(a) for n, a in self.v.items()}, self.C
        s = dict(x=f64(x), ctx=f64(ctx))
        s["qkv"] = norm_fwd(s["x"], v["g1"], v["b1"]) @ w["wqkv"].T
        s["o1"] = self.attn(s["qkv"][..., :C], s["qkv"][..., C:2 * C], s["qkv"][..., 2 * C:], False)
        s["x1"] = s["x"] + s["o1"] @ w["wo"].T
        s["q2"] = norm_fwd(s["x1"], v["g2"], v["b2"]) @ w["wq2"].T
        s["k2"], s["v2"] = s["ctx"] @ w["wk2"].T, s["ctx"] @ w["wv2"].T
        s["o2"] = self.attn(s["q2"], s["k2"], s["v2"], True)
        s["x2"] = s["x1"] + s["o2"] @ w["wo2"].T
        s["h"] = norm_fwd(s["x2"], v["g3"], v["b3"]) @ w["w1"].T + v["bias1"]
        s["y"] = s["x2"] + (s["h"][..., :self.F] * gelu(s["h"][..., self.F:])) @ w["w2"].T
        return s

    def backward(self, s, dy):
        w, v, C, F = self.w, {n: f64(a) for n, a in self.v.items()}, self.C, self.F
        g = {}
        dh = np.concatenate(bwd_ref.geglu_parts(s["h"][..., :F], s["h"][..., F:], dy @ w["w2"]), -1)
        dn, g["dg3"], g["db3"] = norm_bwd(s["x2"], v["g3"], dh @ w["w1"])
        dx2 = dy + dn
        dq, dk, dv = self.attn_bwd(s["q2"], s["k2"], s["v2"], dx2 @ w["wo2"], True)
        g["dctx"] = dk @ w["wk2"] + dv @ w["wv2"]
        dn, g["dg2"], g["db2"] = norm_bwd(s["x1"], v["g2"], dq @ w["wq2"])
        dx1 = dx2 + dn
        d = self.attn_bwd(s["qkv"][..., :C], s["qkv"][..., C:2 * C], s["qkv"][..., 2 * C:], dx1 @ w["wo"], False)
        dn, g["dg1"], g["db1"] = norm_bwd(s["x"], v["g1"], np.concatenate(d, -1) @ w["wqkv"])
        g["dx"] = dx1 + dn
        return g


class Work:
    """A workspace as the wrappers take it."""

    def __init__(self, handle, n):
        self.value, self.nbytes, self.handle = handle.ptr, n, handle


class Device:
    """The block's operands on a backend and its backward pass there, every gradient between the operators fp32. stages:
    what the forward pass left (x, x1, x2, qkv, o1, q2, k2, v2, o2, h), in fp32."""

    def __init__(self, be, ops, blk, stages):
        self.be, self.ops, self.blk = be, ops, blk
        b = blk
        R, Rc, C, F = b.batch * b.T, b.batch * b.Tc, b.C, b.F
        self.R, self.Rc = R, Rc
        put = lambda a: be.buf(np.ascontiguousarray(a).reshape(-1))  # noqa: E731
        self.w = {n: put(a) for n, a in b.raw.items()}
        self.v = {n: put(a) for n, a in b.v.items()}
        self.s = {n: put(np.asarray(a, np.float32)) for n, a in stages.items() if n != "y"}
        self.dy, self.lens = put(b.dy), put(np.asarray(b.lens, np.int32))
        n = dict(dG=R * F, dh=R * 2 * F, dn3=R * C, dx2=R * C, do2=R * C, dq2=R * C, dk2=Rc * C, dv2=Rc * C, dn2=R * C, dx1=R * C,
                 do1=R * C, dqkv=R * 3 * C, dn1=R * C, dx=R * C, dctx=Rc * b.Cc)
        n.update({k + str(i): C for k in ("dg", "db") for i in (1, 2, 3)})
        self.n = n
        self.out = {k: be.buf(np.full(m, bwd_ref.SENTINEL, np.float32)) for k, m in n.items()}
        need = max(ops.gemm_bwd_workspace_bytes(R, 2 * F, C), ops.gemm_bwd_workspace_bytes(R, 3 * C, C), ops.gemm_bwd_workspace_bytes(R, C, F),
                   ops.gemm_bwd_workspace_bytes(Rc, C, b.Cc), ops.gemm_bwd_workspace_bytes(R, C, C), ops.layernorm_bwd_ws_bytes(R, C),
                   ops.fused_attention_bwd_ws_bytes(batch=b.batch, Tq=b.T, Tk=b.T, C=C, heads=b.heads),
                   ops.fused_attention_bwd_ws_bytes(batch=b.batch, Tq=b.T, Tk=b.Tc, C=C, heads=b.heads))
        self.ws = Work(be.buf(np.full(need, 0xff, np.uint8)), need)  # one for all of them, in turn

    def backward(self, stream=None):
        o, b, ops, ws = {k: h.ptr for k, h in self.out.items()}, self.blk, self.ops, self.ws
        w, v, s = ({k: h.ptr for k, h in d.items()} for d in (self.w, self.v, self.s))
        R, Rc, C, F = self.R, self.Rc, b.C, b.F

        def linear(dc, wt, da, M, N, K, **kw):
            ops.gemm_nt_q8_0_bwd(dc, w[wt], da, M, N, K, workspace=ws, stream=stream, **kw)

        def norm(i, x, dn, res, dx):
            ops.layernorm_bwd(x, v[f"g{i}"], dn, dx, o[f"dg{i}"], o[f"db{i}"], ws, R, C, res=res, stream=stream)

        linear(self.dy.ptr, "w2", o["dG"], R, C, F)
        ops.geglu_bwd(s["h"], o["dG"], o["dh"], R, F, stream=stream)
        linear(o["dh"], "w1", o["dn3"], R, 2 * F, C)
        norm(3, s["x2"], o["dn3"], self.dy.ptr, o["dx2"])
        linear(o["dx2"], "wo2", o["do2"], R, C, C)
        ops.fused_attention_bwd(s["q2"], s["k2"], s["v2"], s["o2"], o["do2"], o["dq2"], o["dk2"], o["dv2"], ws, batch=b.batch, Tq=b.T,
                                Tk=b.Tc, C=C, heads=b.heads, kv_len=self.lens.ptr, stream=stream)
        linear(o["dk2"], "wk2", o["dctx"], Rc, C, b.Cc)
        linear(o["dv2"], "wv2", o["dctx"], Rc, C, b.Cc, mode=1)
        linear(o["dq2"], "wq2", o["dn2"], R, C, C)
        norm(2, s["x1"], o["dn2"], o["dx2"], o["dx1"])
        linear(o["dx1"], "wo", o["do1"], R, C, C)
        q, d = s["qkv"], o["dqkv"]
        ops.fused_attention_bwd(q, q + 4 * C, q + 8 * C, s["o1"], o["do1"], d, d + 4 * C, d + 8 * C, ws, batch=b.batch, Tq=b.T, Tk=b.T, C=C,
                                heads=b.heads, ldq=3 * C, ldk=3 * C, ldv=3 * C, lddq=3 * C, lddk=3 * C, lddv=3 * C, stream=stream)
        linear(o["dqkv"], "wqkv", o["dn1"], R, 3 * C, C)
        norm(1, s["x"], o["dn1"], o["dx1"], o["dx"])

    def results(self):
        b = self.blk
        r = {k: self.be.get(self.out[k], np.float32, self.n[k]) for k in RESULTS}
        r["dx"] = r["dx"].reshape(b.batch, b.T, b.C)
        r["dctx"] = r["dctx"].reshape(b.batch, b.Tc, b.Cc)
        return r


# Each operator leaves 8 x 2^-22 of its result at most in the mean (test bounds of each alone), and passes on what its inputs
# carry through the same linear map as the gradient itself: in the mean the same share of it; four times that for the maps
# that take more away from the gradient than from an error (LayerNorm's projections, dP - delta). Twelve operators on the
# longest path; the stored stages' own rounding (u each) is far below.
BLOCK_REL = 12 * 8 * 2.0 ** -22 * 4


def check_block(blk, got, want):
    for k in RESULTS:
        assert np.all(np.isfinite(got[k])), k
        rel = np.linalg.norm(f64(got[k]) - want[k]) / np.linalg.norm(want[k])
        assert rel <= BLOCK_REL, f"{k}: relative error {rel:.3e} > {BLOCK_REL:.3e}"
    for i, n in enumerate(blk.lens):
        assert np.all(got["dctx"][i, n:] == 0), "a context token past its row's length has a gradient"


def slope(blk, dx, dctx, eps):
    """d/dt <dy, block(x + t dx, ctx + t dctx)> at 0 by central differences in 64 bits."""
    dy = f64(blk.dy)

    def f(t):
        return float((blk.forward(f64(blk.x) + t * dx, f64(blk.ctx) + t * dctx)["y"] * dy).sum())

    return (f(eps) - f(-eps)) / (2 * eps)


def check_differences(blk, got, tol):
    """The slope along the gradient itself is its length, and along any other direction its product with it. Of unit
    directions over some 30000 inputs (each input moves by 2^-8 eps) the third derivative's share is under eps^2."""
    g = (f64(got["dx"]), f64(got["dctx"]))
    size = math.sqrt(sum(float((a * a).sum()) for a in g))
    r = rng_of(3)
    for d in (g, [r.standard_normal(a.shape) for a in g]):
        n = math.sqrt(sum(float((a * a).sum()) for a in d))
        d = [a / n for a in d]
        want = slope(blk, *d, 2.0 ** -7)
        have = sum(float((a * b).sum()) for a, b in zip(g, d))
        assert abs(have - want) <= (tol + 2.0 ** -14) * size, (have, want, size)


def block(be, seed=11):
    """bwd_ref's form of a case: the whole backward pass on a backend, twice."""
    from sdvk_amd import ops

    blk = Block(seed)
    stages = blk.forward(blk.x, blk.ctx)
    dev = Device(be, ops, blk, stages)
    dev.backward()
    got = dev.results()
    check_block(blk, got, blk.backward(stages, f64(blk.dy)))
    check_differences(blk, got, BLOCK_REL)
    dev.backward()
    again = dev.results()
    assert all(np.array_equal(got[k].view(np.uint32), again[k].view(np.uint32)) for k in RESULTS), "a second pass gave other bits"


def feed_forward_f16(be, seed=12):
    """The feed-forward half in fp16, its projection recomputed: n3 = LayerNorm, dG = dy W2, dH from (n3, W1, dG) in one
    GEMM, dn3 = dH W1, dx = dy + LayerNorm's gradient."""
    from sdvk_amd import ops

    blk = Block(seed)
    R, C, F = blk.batch * blk.T, blk.C, blk.F
    x = f64(blk.x).reshape(R, C)
    v = {n: f64(a) for n, a in blk.v.items()}
    dy16 = (blk.dy * 256).astype(np.float16).reshape(R, C)
    n3 = norm_fwd(x, v["g3"], v["b3"])
    put = lambda a: be.buf(np.ascontiguousarray(a).reshape(-1))  # noqa: E731
    bx, bn, bdy = put(blk.x), put(n3.astype(np.float16)), put(dy16)
    w1, w2, b1, g3 = put(blk.raw["w1"]), put(blk.raw["w2"]), put(blk.v["bias1"]), put(blk.v["g3"])
    dG, dH, dn = (be.buf(np.full(n, 7, np.float16)) for n in (R * F, R * 2 * F, R * C))
    dx, dg, db = (be.buf(np.full(n, 7, np.float32)) for n in (R * C, C, C))
    need = max(ops.gemm_bwd_workspace_bytes(R, C, F, dtype=ops.MI_F16), ops.gemm_bwd_workspace_bytes(R, 2 * F, C, dtype=ops.MI_F16),
               ops.layernorm_bwd_ws_bytes(R, C))
    ws = Work(be.buf(np.full(need, 0xff, np.uint8)), need)
    ops.gemm_nt_q8_0_bwd(bdy.ptr, w2.ptr, dG.ptr, R, C, F, dtype=ops.MI_F16, workspace=ws)
    ops.gemm_nt_q8_0_geglu_bwd(bn.ptr, w1.ptr, dG.ptr, dH.ptr, R, F, C, bias=b1.ptr)
    ops.gemm_nt_q8_0_bwd(dH.ptr, w1.ptr, dn.ptr, R, 2 * F, C, dtype=ops.MI_F16, workspace=ws)
    ops.layernorm_bwd(bx.ptr, g3.ptr, dn.ptr, dx.ptr, dg.ptr, db.ptr, ws, R, C, dy_dtype=ops.MI_F16)
    got = f64(be.get(dx, np.float32, R * C)).reshape(R, C)
    h = n3 @ blk.w["w1"].T + v["bias1"]
    dh = np.concatenate(bwd_ref.geglu_parts(h[:, :F], h[:, F:], f64(dy16) @ blk.w["w2"]), -1)
    want, wg, wb = norm_bwd(x, v["g3"], dh @ blk.w["w1"])
    # fp16 roundings, H / sqrt 3 each at most in the mean: dy W2's weights and result, n3, W1's weights (twice), dH, dn3; the
    # same factor of four as above
    tol = 4 * math.sqrt(7) * H / math.sqrt(3)
    for a, b in ((got, want), (f64(be.get(dg, np.float32, C)), wg), (f64(be.get(db, np.float32, C)), wb)):
        rel = np.linalg.norm(a - b) / np.linalg.norm(b)
        assert rel <= tol, (rel, tol)
    # along the gradient, against differences of the 64-bit forward pass
    d = got / np.linalg.norm(got)

    def f(t):
        hh = norm_fwd(x + t * d, v["g3"], v["b3"]) @ blk.w["w1"].T + v["bias1"]
        return float(((hh[:, :F] * gelu(hh[:, F:])) @ blk.w["w2"].T * f64(dy16)).sum())

    e = 2.0 ** -7
    assert abs((f(e) - f(-e)) / (2 * e) - np.linalg.norm(got)) <= (tol + 2.0 ** -14) * np.linalg.norm(got)


OPS = {"block": block, "feed_forward_f16": feed_forward_f16}
