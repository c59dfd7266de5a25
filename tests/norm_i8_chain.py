"""The operators run together, as a UNet's transformer would use them around its blocks: GroupNorm into 8-bit rows, proj_in, a feed-forward
in 8 bits (LayerNorm, quantiser, product, GEGLU, quantiser, product onto the residual), quantiser, proj_out onto the input; and
backwards, from the gradient of a Q8_0 linear behind a GroupNorm with SiLU to its input and weights. Nothing is read back in between;
then every stage is checked against 64 bits from the inputs that it had, and the whole against the float computation."""
from __future__ import annotations

import numpy as np

import norm_i8_ref as ref
from bwd_block import Work, gelu, norm_bwd  # noqa: F401
from bwd_ref import H, SENTINEL, TINY16, U, check, f64, q8_blocks, rng_of, store_err

EPS = 1e-5


def weight_codes(w):
    return ref.codes_of(w.astype(np.float32))


class Chain:
    def __init__(self, be, ops, seed=5, B=2, P=70, C=128, G=32, F=160, N=96):
        r = rng_of(seed)
        self.be, self.ops, self.B, self.P, self.C, self.G, self.F, self.N, self.R = be, ops, B, P, C, G, F, N, B * P
        R = self.R
        self.x = ref.pixels_of(r, B, P, C, 0.5, 0.0).astype(np.float32)
        self.vec = {n: (1 + 0.2 * r.standard_normal(C)).astype(np.float32) for n in ("gg", "lg")}
        self.vec |= {n: (0.2 * r.standard_normal(k)).astype(np.float32) for n, k in (("gb", C), ("lb", C), ("b_in", C), ("b_up", 2 * F), ("b_down", C), ("b_out", C))}
        self.w = {n: r.standard_normal(s) / np.sqrt(s[1]) for n, s in (("in", (C, C)), ("up", (2 * F, C)), ("down", (C, F)), ("out", (C, C)))}
        self.codes = {n: weight_codes(w) for n, w in self.w.items()}
        self.x16 = ref.pixels_of(r, B, P, C, -0.3, 0.0).astype(np.float16)
        self.dC = (0.5 * r.standard_normal((R, N))).astype(np.float16)
        self.skip = (0.5 * r.standard_normal((B, P, C))).astype(np.float16)
        self.raw, self.wq = q8_blocks(r.standard_normal((N, C)) * 0.05)
        put = lambda a: be.buf(np.ascontiguousarray(a).reshape(-1))  # noqa: E731
        self.dev = {"x": put(self.x), "x16": put(self.x16), "dC": put(self.dC), "skip": put(self.skip), "raw": put(self.raw)}
        self.dev |= {n: put(v) for n, v in self.vec.items()}
        for n, (q, s) in self.codes.items():
            self.dev["w_" + n], self.dev["s_" + n] = put(q), put(s)
        f32, f16, i8 = np.float32, np.float16, np.int8
        self.kinds = dict(q0=(R * C, i8), s0=(R, f32), t=(R * C, f32), ln=(R * C, f16), q1=(R * C, i8), s1=(R, f32), h=(R * 2 * F, f32), g=(R * F, f16), q2=(R * F, i8),
                          s2=(R, f32), q3=(R * C, i8), s3=(R, f32), y=(R * C, f32), act=(R * C, f16), stats=(B * G * 4, f32), dn=(R * C, f16), dx=(R * C, f16),
                          dgamma=(C, f32), dbeta=(C, f32))
        self.out = {n: be.buf(np.full(k, SENTINEL).astype(t)) for n, (k, t) in self.kinds.items()}
        size = dict(batch=B, pixels=P, C=C, groups=G)
        self.size = size
        need = max(ops.groupnorm_ws_bytes(**size), ops.groupnorm_bwd_ws_bytes(**size), ops.gemm_bwd_workspace_bytes(R, N, C, dtype=ops.MI_F16))
        self.ws = Work(be.buf(np.full(need, 0xff, np.uint8)), need)  # one for all of them, in turn
        # y starts as the input: proj_out adds to it
        self.copy_y = put(self.x)

    def run(self, stream=None):
        """y must hold x: `reset` does that."""
        o, ops, R, C, F, s = self.ops, self.ops, self.R, self.C, self.F, stream
        d = {n: h.ptr for n, h in {**self.dev, **self.out}.items()}
        o.groupnorm(d["x"], d["gg"], d["gb"], d["q0"], self.ws, y_dtype=ops.MI_I8, y_scale=d["s0"], eps=1e-6, stream=s, **self.size)
        o.gemm_nt_i8(d["q0"], d["s0"], d["w_in"], d["s_in"], d["t"], R, C, C, bias=d["b_in"], stream=s)
        o.layernorm_f16(d["t"], d["lg"], d["lb"], d["ln"], R, C, stream=s)
        o.quantize_rows_i8(d["ln"], d["q1"], d["s1"], R, C, dtype=ops.MI_F16, stream=s)
        o.gemm_nt_i8(d["q1"], d["s1"], d["w_up"], d["s_up"], d["h"], R, 2 * F, C, bias=d["b_up"], stream=s)
        o.geglu_f16(d["h"], d["g"], R, F, stream=s)
        o.quantize_rows_i8(d["g"], d["q2"], d["s2"], R, F, dtype=ops.MI_F16, stream=s)
        o.gemm_nt_i8(d["q2"], d["s2"], d["w_down"], d["s_down"], d["t"], R, C, F, bias=d["b_down"], mode=2, stream=s)
        o.quantize_rows_i8(d["t"], d["q3"], d["s3"], R, C, stream=s)
        o.gemm_nt_i8(d["q3"], d["s3"], d["w_out"], d["s_out"], d["y"], R, C, C, bias=d["b_out"], mode=2, stream=s)
        o.groupnorm(d["x16"], d["gg"], d["gb"], d["act"], self.ws, act=ops.MI_ACT_SILU, x_dtype=ops.MI_F16, y_dtype=ops.MI_F16, stats=d["stats"], stream=s, **self.size)
        o.gemm_nt_q8_0_bwd(d["dC"], d["raw"], d["dn"], R, self.N, C, dtype=ops.MI_F16, workspace=self.ws, stream=s)
        o.groupnorm_bwd(d["x16"], d["gg"], d["gb"], d["dn"], d["dx"], d["dgamma"], d["dbeta"], self.ws, act=ops.MI_ACT_SILU, x_dtype=ops.MI_F16, dy_dtype=ops.MI_F16,
                        res=d["skip"], stats=d["stats"], stream=s, **self.size)

    def results(self):
        return {n: self.be.get(self.out[n], t, k) for n, (k, t) in self.kinds.items()}

    def reset(self, put):
        """Every output and the workspace as before a run: put(handle, array)."""
        for n, (k, t) in self.kinds.items():
            put(self.out[n], np.full(k, SENTINEL).astype(t) if n != "y" else self.x.reshape(-1))
        put(self.ws.handle, np.full(self.ws.nbytes, 0xff, np.uint8))

    # ---- checks ----

    def linear(self, q, s, name, bias, old=None):
        """(want, bound) of a product's result in fp32."""
        wq, ws = self.codes[name]
        part = (f64(q) @ f64(wq).T) * f64(s)[:, None] * f64(ws)
        want = part + f64(self.vec[bias])
        tol = 3.01 * U * np.abs(part) + U * np.abs(want)
        if old is not None:
            want = want + old
            tol = tol + U * np.abs(want)
        return want, tol + U * np.abs(want) + 1e-37

    def check(self, got):
        R, C, F, B, P = self.R, self.C, self.F, self.B, self.P
        m = {n: got[n].reshape(R, -1) for n in ("q0", "t", "ln", "q1", "h", "g", "q2", "q3", "y")}
        # GroupNorm's rows
        q = ref.Group(self.x, self.G, 1e-6)
        want, e = (a.reshape(R, C) for a in ref.forward64(q, self.vec["gg"], self.vec["gb"], 0, (B, P, C)))
        sc = f64(got["s0"])[:, None]
        check(sc, np.abs(want).max(1, keepdims=True) / 127, e.max(1, keepdims=True) / 127 + sc * 2 * U, "entry scale")
        check(f64(m["q0"]) * sc, want, 0.5 * sc * (1 + 1e-6) + e, "entry codes")
        # proj_in, from the codes; t itself has been added to since
        t, et = self.linear(m["q0"], got["s0"], "in", "b_in")
        xc = t - t.mean(1, keepdims=True)
        inv = 1 / np.sqrt((xc * xc).mean(1, keepdims=True) + EPS)
        ln = xc * inv * f64(self.vec["lg"]) + f64(self.vec["lb"])
        e_ln = (et + et.mean(1, keepdims=True)) * inv * np.abs(f64(self.vec["lg"])) * 2 + (C / 64 + 24) * U * (np.abs(xc * inv) * 2 + 2 + np.abs(ln))
        check(m["ln"], ln, e_ln + store_err(ln, "f16") * 1.01, "LayerNorm")
        for n, src, cols in (("1", m["ln"], C), ("2", m["g"], F), ("3", m["t"], C)):
            qq, ss = ref.codes_of(src.astype(np.float32))
            assert np.array_equal(qq, m["q" + n]) and np.array_equal(ss, got["s" + n]), f"codes {n}"
        h, eh = self.linear(m["q1"], got["s1"], "up", "b_up")
        check(m["h"], h, eh, "FF-up")
        v, gate = f64(m["h"][:, :F]), f64(m["h"][:, F:])
        g = v * gelu(gate)
        check(m["g"], g, np.abs(v) * (np.abs(gate) * 4e-7 + 4e-7) + store_err(g, "f16") * 1.01, "GEGLU")
        t2, et2 = self.linear(m["q2"], got["s2"], "down", "b_down", t)
        check(m["t"], t2, et2 + et, "FF-down onto the residual")
        y, ey = self.linear(m["q3"], got["s3"], "out", "b_out", f64(self.x).reshape(R, C))
        check(m["y"], y, ey, "proj_out onto the input")
        self.check_whole(got, want)
        # backwards
        x16 = self.x16
        q = ref.Group(x16, self.G, EPS)
        want, e = ref.forward64(q, self.vec["gg"], self.vec["gb"], 1, (B, P, C))
        check(got["act"].reshape(B, P, C), want, e + store_err(want, "f16") * 1.01, "GroupNorm SiLU")
        dn = f64(self.dC) @ self.wq
        mag = np.abs(f64(self.dC)) @ np.abs(self.wq)
        check(got["dn"].reshape(R, C), dn, mag * (H * 1.01 + (self.N + 8) * U) + np.abs(f64(self.dC)).sum(1, keepdims=True) * TINY16 + store_err(dn, "f16") * 1.01, "dn")
        (dx, e1), (dg, e2), (db, e3) = ref.backward64(q, got["dn"].reshape(B, P, C), self.vec["gg"], self.vec["gb"], 1, self.skip)
        check(got["dx"].reshape(B, P, C), dx, e1 + store_err(dx, "f16") * 1.01, "dx")
        check(got["dgamma"], dg, e2, "dgamma")
        check(got["dbeta"], db, e3, "dbeta")

    def check_whole(self, got, n0):
        """y against the computation without codes. A code is off by half a step at most, 1 / sqrt 12 of one in the mean: of a row's (or
        channel's) values that is scale / (sqrt 12 rms). Eight tensors in codes, each passing on what it has to y about as
        it passes on the values themselves; a factor of three for the maps that take more from a value than from an error."""
        v, w = self.vec, self.w
        t = n0 @ w["in"].T + v["b_in"]
        xc = t - t.mean(1, keepdims=True)
        ln = xc / np.sqrt((xc * xc).mean(1, keepdims=True) + EPS) * v["lg"] + v["lb"]
        h = ln @ w["up"].T + v["b_up"]
        g = h[:, :self.F] * gelu(h[:, self.F:])
        t = t + g @ w["down"].T + v["b_down"]
        d = t @ w["out"].T + v["b_out"]
        noise = 0.0
        for a in (n0, ln, g, t, *w.values()):
            noise += float(np.mean((np.abs(a).max(1) / 127 / np.sqrt(12)) ** 2 / (a ** 2).mean(1)))
        have = f64(got["y"]).reshape(self.R, self.C) - f64(self.x).reshape(self.R, self.C)
        rel = np.linalg.norm(have - d) / np.linalg.norm(d)
        assert rel <= 3 * np.sqrt(noise), (rel, np.sqrt(noise))


def chain(be, **kw):
    """A case of norm_i8_ref's form: the whole run on a backend."""
    from sdvk_amd import ops

    c = Chain(be, ops, **kw)
    c.out["y"] = c.copy_y
    c.run()
    c.check(c.results())


OPS = {"chain": chain}
