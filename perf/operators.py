"""The backward passes that fine-tuning an SDXL UNet on frozen Q8_0 weights calls, as measurable cases.

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run` is one pass through an operator, `work`
the bytes and operations that the pass cannot do without, `exact` the same result in 64 bits from the operator's
definition. `own` chooses what `run` does: elementary torch operations in 32 bits, rounded once at the end, or the
package's entry points (sdvk_amd.ops), which take addresses: the library is then bound to the HIP runtime that torch
has loaded, so that there is one runtime and one default stream.

Sizes: an image has sides of 512 to 1536 pixels in steps of 64, a megapixel at most; a UNet level of 640 channels has
(H / 16) x (W / 16) tokens and one of 1280 channels (H / 32) x (W / 32), times one or two rows of a batch. The context
is 77 tokens a prompt chunk of 2048 channels. Gradients in fp16 are of the size a loss scale gives them, those in
fp32 are not scaled.
"""
from __future__ import annotations

import math
from pathlib import Path

import torch

own = False

DEV = "cuda"
CTX_TOKENS, CTX_CHANNELS = 77, 2048
TYPES = {"f16": torch.float16, "f32": torch.float32}
GRAD_STD = {"f16": 0.5, "f32": 1e-3}
LINEARS = [(640, 640), (1280, 1280), (1920, 640), (640, 2560), (1280, 5120), (5120, 640), (10240, 1280), (1280, 2048)]


def listed():
    return [
        # ---- attention, from its inputs and its output to the gradients of q, k and v
        # self-attention of the 640-channel level at 1024 x 1024, fp16, a batch of two
        dict(name="attn_f16_self_2x10x4096", kind="attn", type="f16", batch=2, heads=10, hd=64, Tq=4096, Tk=4096, causal=False, masked=False),
        # cross-attention of the 1280-channel level on prompts padded to 77 tokens
        dict(name="attn_f16_cross_2x20x1024x77", kind="attn", type="f16", batch=2, heads=20, hd=64, Tq=1024, Tk=77, causal=False, masked=True),
        # the fp32 attention entry's own types at 768 x 768, one image
        dict(name="attn_f32_self_10x2304", kind="attn", type="f32", batch=1, heads=10, hd=64, Tq=2304, Tk=2304, causal=False, masked=False),
        # a text encoder's causal self-attention of one prompt: a call where latency counts
        dict(name="attn_f32_causal_12x77", kind="attn", type="f32", batch=1, heads=12, hd=64, Tq=77, Tk=77, causal=True, masked=False),
        # ---- LayerNorm: gradients of x (with the residual's added) and of the weights
        # the 640-channel level at 1024 x 1024, both images, fp32 gradient
        dict(name="norm_8192x640", kind="norm", type="f32", rows=8192, d=640, affine=True, residual=True),
        # a text encoder's norm over one prompt, fp16 gradient from the projections
        dict(name="norm_f16_77x768", kind="norm", type="f16", rows=77, d=768, affine=True, residual=True),
        # ---- GEGLU: from the projection that the forward pass kept, or from the feed-forward's input
        # 1280-channel level at 1024 x 1024, both images, fp32, projection kept
        dict(name="geglu_f32_2048x5120", kind="geglu", type="f32", rows=2048, F=5120),
        # 1280-channel level at 832 x 1216 (2 x 26 x 38 tokens), projections recomputed from fp16 activations
        dict(name="geglu_gemm_1976x5120x1280", kind="geglu_gemm", M=1976, F=5120, K=1280, bias=True),
        # 640-channel level at 512 x 512 (32 x 32 tokens), one image
        dict(name="geglu_gemm_1024x2560x640", kind="geglu_gemm", M=1024, F=2560, K=640, bias=True),
        # ---- a frozen Q8_0 linear: the gradient of its input
        # a ResBlock's time-embedding projection, a batch of two: the smallest
        dict(name="linear_f32_2x1280x1280", kind="linear", type="f32", M=2, N=1280, K=1280),
        # FF-down at 1024 x 1024, fp16
        dict(name="linear_f16_2048x1280x5120", kind="linear", type="f16", M=2048, N=1280, K=5120),
        # an attention projection at 768 x 768 (2 x 24 x 24 tokens), fp32
        dict(name="linear_f32_1152x1280x1280", kind="linear", type="f32", M=1152, N=1280, K=1280),
    ]


def draw(rng):
    h, w = 64 * rng.randint(8, 24), 64 * rng.randint(8, 24)
    while h * w > 1024 * 1024:  # trained sizes: a megapixel at most
        h, w = 64 * rng.randint(8, 24), 64 * rng.randint(8, 24)
    rows = rng.choice([1, 2, 2])
    C = rng.choice([640, 1280])
    tokens = (h // 16) * (w // 16) if C == 640 else (h // 32) * (w // 32)
    typ = rng.choice(["f16", "f16", "f32"])
    kind = rng.choice(["self", "cross", "attn", "norm", "geglu", "geglu_gemm", "geglu_gemm", "linear", "linear"])
    if kind == "self":
        return dict(kind="attn", type=typ, batch=rows, heads=C // 64, hd=64, Tq=tokens, Tk=tokens, causal=False, masked=False)
    if kind == "cross":
        return dict(kind="attn", type=typ, batch=rows, heads=C // 64, hd=64, Tq=tokens, Tk=CTX_TOKENS * rng.randint(1, 3),
                    causal=False, masked=rng.random() < 0.7)
    if kind == "attn":  # any lengths and head widths, causal or padded
        Tq = int(2 ** rng.uniform(0, 11))
        causal = rng.random() < 0.4
        return dict(kind="attn", type=typ, batch=rng.randint(1, 3), heads=rng.randint(1, 12), hd=rng.choice([64, 64, 40, 32, 20]),
                    Tq=Tq, Tk=Tq if causal else int(2 ** rng.uniform(0, 11)), causal=causal, masked=rng.random() < 0.5)
    if kind == "norm":
        n = rows * tokens if rng.random() < 0.6 else int(2 ** rng.uniform(0, 12))
        return dict(kind="norm", type=typ, rows=n, d=rng.choice([C, C, 320, 768, 1001]), affine=rng.random() < 0.8, residual=rng.random() < 0.7)
    if kind == "geglu":
        return dict(kind="geglu", type=typ, rows=rows * tokens if rng.random() < 0.6 else int(2 ** rng.uniform(0, 11)), F=rng.choice([4 * C, 4 * C, 1277]))
    if kind == "geglu_gemm":
        return dict(kind="geglu_gemm", M=rows * tokens if rng.random() < 0.7 else int(2 ** rng.uniform(0, 11)), F=4 * C, K=C, bias=rng.random() < 0.8)
    N, K = rng.choice(LINEARS)
    M = rng.choice([rng.randint(1, 16), CTX_TOKENS * rng.randint(1, 4), rows * tokens, rows * tokens])
    M = min(M, 2 ** 37 // (2 * N * K))  # a pass of no more work than the largest listed one
    return dict(kind="linear", type=typ, M=M, N=N, K=K)


# ------------------------------------------------------------------ inputs --

def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0):
    x = torch.empty(*shape, device=DEV).normal_(generator=g)
    return x.mul_(std) if std != 1.0 else x


def blocks_of(w):
    """The 34-byte GGUF Q8_0 blocks of an fp32 weight, as bytes."""
    b = w.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    q = torch.round(b * torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))).clamp(-127, 127).to(torch.int8)
    return torch.cat([(amax / 127.0).to(torch.float16).view(torch.uint8), q.view(torch.uint8)], 1).reshape(-1)


def attn_inputs(c, seed):
    g = generator(seed)
    dt, C = TYPES[c["type"]], c["heads"] * c["hd"]
    q, k, v = (normal(g, c["batch"], t, C).to(dt) for t in (c["Tq"], c["Tk"], c["Tk"]))
    do = normal(g, c["batch"], c["Tq"], C, std=GRAD_STD[c["type"]]).to(dt)
    lens = torch.randint(1, c["Tk"] + 1, (c["batch"],), generator=g, device=DEV, dtype=torch.int32) if c["masked"] else None
    return dict(q=q, k=k, v=v, do=do, lens=lens)


def norm_inputs(c, seed):
    g = generator(seed)
    rows, d = c["rows"], c["d"]
    x = normal(g, rows, d, std=2.0) + 0.5
    s = dict(x=x, dy=normal(g, rows, d, std=GRAD_STD[c["type"]]).to(TYPES[c["type"]]),
             gamma=1 + normal(g, d, std=0.2) if c["affine"] else None,
             res=normal(g, rows, d, std=GRAD_STD[c["type"]]) if c["residual"] else None)
    return s


def geglu_inputs(c, seed):
    g = generator(seed)
    return dict(h=normal(g, c["rows"], 2 * c["F"], std=1.5),
                dy=normal(g, c["rows"], c["F"], std=GRAD_STD[c["type"]]).to(TYPES[c["type"]]))


def geglu_gemm_inputs(c, seed):
    g = generator(seed)
    M, F, K = c["M"], c["F"], c["K"]
    return dict(A=normal(g, M, K).half(), W=blocks_of(normal(g, 2 * F, K, std=0.02)),
                bias=normal(g, 2 * F, std=0.02) if c["bias"] else None, dG=normal(g, M, F, std=GRAD_STD["f16"]).half())


def linear_inputs(c, seed):
    g = generator(seed)
    return dict(dC=normal(g, c["M"], c["N"], std=GRAD_STD[c["type"]]).to(TYPES[c["type"]]),
                W=blocks_of(normal(g, c["N"], c["K"], std=0.02)))


INPUTS = {"attn": attn_inputs, "norm": norm_inputs, "geglu": geglu_inputs, "geglu_gemm": geglu_gemm_inputs, "linear": linear_inputs}


def heads_of(x, heads):
    """[batch, heads, T, hd] in 32 bits of a [batch, T, heads * hd] tensor."""
    b, t, c = x.shape
    return x.float().reshape(b, t, heads, c // heads).transpose(1, 2).contiguous()


def seen(c, lens):
    """Which keys a query sees: [batch or 1, 1, Tq or 1, Tk], or None for all."""
    keys = torch.arange(c["Tk"], device=DEV)
    m = None
    if lens is not None:
        m = (keys[None, :] < lens[:, None])[:, None, None, :]
    if c["causal"]:
        up = (keys[None, :] <= torch.arange(c["Tq"], device=DEV)[:, None])[None, None]
        m = up if m is None else m & up
    return m


def probabilities(q, k, m):
    """Softmax over the seen keys in 32 bits; rows that see none are zero."""
    p = q @ k.transpose(-1, -2)
    p *= 1.0 / math.sqrt(q.shape[-1])
    if m is not None:
        p = torch.where(m, p, torch.full_like(p, -math.inf))
    top = p.amax(-1, keepdim=True)
    p -= torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p.exp_()
    total = p.sum(-1, keepdim=True)
    return p * torch.where(total > 0, 1.0 / total, torch.zeros_like(total))


def prepare(case, seed):
    c = case
    s = INPUTS[c["kind"]](c, seed)
    s["case"] = c
    if c["kind"] == "attn":
        # the forward pass's output, which a training step has kept
        q, k, v = (heads_of(s[n], c["heads"]) for n in ("q", "k", "v"))
        o = probabilities(q, k, seen(c, s["lens"])) @ v
        s["o"] = o.transpose(1, 2).reshape(s["q"].shape).to(TYPES[c["type"]])
        s["out"] = [torch.empty_like(s[n]) for n in ("q", "k", "v")]
    elif c["kind"] == "norm":
        s["out"] = [torch.empty_like(s["x"])] + [torch.empty(c["d"], device=DEV) for _ in range(2 if c["affine"] else 0)]
    elif c["kind"] == "geglu":
        s["out"] = [torch.empty(c["rows"], 2 * c["F"], device=DEV, dtype=TYPES[c["type"]])]
    elif c["kind"] == "geglu_gemm":
        s["out"] = [torch.empty(c["M"], 2 * c["F"], device=DEV, dtype=torch.float16)]
    else:
        s["out"] = [torch.empty(c["M"], c["K"], device=DEV, dtype=TYPES[c["type"]])]
    return s


# -------------------------------------------------------------- plain form --

def weight(raw, n, k):
    """32-bit values of a weight of n rows of 34-byte blocks."""
    b = raw.reshape(-1, 34)
    d = b[:, :2].contiguous().view(torch.float16).float()
    return (b[:, 2:].contiguous().view(torch.int8).float() * d).reshape(n, k)


def gelu_and_slope(x):
    half = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x * half, half + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def attn_plain(s, c):
    q, k, v, do = (heads_of(s[n], c["heads"]) for n in ("q", "k", "v", "do"))
    p = probabilities(q, k, seen(c, s["lens"]))
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    ds *= 1.0 / math.sqrt(c["hd"])
    grads = (ds @ k, ds.transpose(-1, -2) @ q, dv)
    return [g.transpose(1, 2).reshape(s[n].shape).to(TYPES[c["type"]]) for g, n in zip(grads, ("q", "k", "v"))]


def norm_plain(s, c):
    x, dy = s["x"], s["dy"].float()
    xc = x - x.mean(-1, keepdim=True)
    inv = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * inv
    g = dy if s["gamma"] is None else dy * s["gamma"]
    dx = inv * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    if s["res"] is not None:
        dx = dx + s["res"]
    return [dx] + ([(dy * xh).sum(0), dy.sum(0)] if c["affine"] else [])


def geglu_plain(s, c):
    F, dy = c["F"], s["dy"].float()
    act, slope = gelu_and_slope(s["h"][:, F:])
    return [torch.cat([dy * act, dy * s["h"][:, :F] * slope], 1).to(TYPES[c["type"]])]


def geglu_gemm_plain(s, c):
    F, dy = c["F"], s["dG"].float()
    h = s["A"].float() @ weight(s["W"], 2 * F, c["K"]).t()
    if s["bias"] is not None:
        h = h + s["bias"]
    act, slope = gelu_and_slope(h[:, F:])
    return [torch.cat([dy * act, dy * h[:, :F] * slope], 1).half()]


def linear_plain(s, c):
    return [(s["dC"].float() @ weight(s["W"], c["N"], c["K"])).to(TYPES[c["type"]])]


PLAIN = {"attn": attn_plain, "norm": norm_plain, "geglu": geglu_plain, "geglu_gemm": geglu_gemm_plain, "linear": linear_plain}


# --------------------------------------------------- the package's operators --

class Buf:
    """A device buffer as the entry points take one: its address and its size in bytes."""

    def __init__(self, nbytes):
        self.t = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=DEV)
        self.value, self.nbytes = self.t.data_ptr(), int(nbytes)


def package():
    """sdvk_amd.ops, bound to torch's HIP runtime: a second one would not know torch's buffers or streams."""
    from sdvk_amd import hip, ops

    if hip._hip is None:
        hip.ROCM = Path(torch.__file__).resolve().parent
    return ops


def address(t):
    return t.data_ptr() if t is not None else None


def kept(s, nbytes):
    """The workspace that a program keeps for the call, made the first time."""
    if "ws" not in s:
        s["ws"] = Buf(nbytes())
    return s["ws"]


def attn_own(ops, s, c):
    dt = ops.MI_F16 if c["type"] == "f16" else ops.MI_F32
    a = dict(batch=c["batch"], Tq=c["Tq"], Tk=c["Tk"], C=c["heads"] * c["hd"], heads=c["heads"], dtype=dt)
    ws = kept(s, lambda: ops.fused_attention_bwd_ws_bytes(**a))
    ops.fused_attention_bwd(*(s[n].data_ptr() for n in ("q", "k", "v", "o", "do")), *(t.data_ptr() for t in s["out"]), ws,
                            causal=c["causal"], kv_len=address(s["lens"]), **a)


def norm_own(ops, s, c):
    ws = kept(s, lambda: ops.layernorm_bwd_ws_bytes(c["rows"], c["d"]))
    out = [t.data_ptr() for t in s["out"]] + [None, None]
    ops.layernorm_bwd(s["x"].data_ptr(), address(s["gamma"]), s["dy"].data_ptr(), out[0], out[1], out[2], ws, c["rows"], c["d"],
                      res=address(s["res"]), dy_dtype=ops.MI_F16 if c["type"] == "f16" else ops.MI_F32)


def geglu_own(ops, s, c):
    ops.geglu_bwd(s["h"].data_ptr(), s["dy"].data_ptr(), s["out"][0].data_ptr(), c["rows"], c["F"],
                  dtype=ops.MI_F16 if c["type"] == "f16" else ops.MI_F32)


def geglu_gemm_own(ops, s, c):
    ops.gemm_nt_q8_0_geglu_bwd(s["A"].data_ptr(), s["W"].data_ptr(), s["dG"].data_ptr(), s["out"][0].data_ptr(), c["M"], c["F"],
                               c["K"], bias=address(s["bias"]))


def linear_own(ops, s, c):
    dt = ops.MI_F16 if c["type"] == "f16" else ops.MI_F32
    ws = kept(s, lambda: ops.gemm_bwd_workspace_bytes(c["M"], c["N"], c["K"], dtype=dt))
    ops.gemm_nt_q8_0_bwd(s["dC"].data_ptr(), s["W"].data_ptr(), s["out"][0].data_ptr(), c["M"], c["N"], c["K"], dtype=dt, workspace=ws)


OWN = {"attn": attn_own, "norm": norm_own, "geglu": geglu_own, "geglu_gemm": geglu_gemm_own, "linear": linear_own}


def run(state):
    s, c = state, state["case"]
    if not own:
        return PLAIN[c["kind"]](s, c)
    OWN[c["kind"]](package(), s, c)
    return s["out"]


# ------------------------------------------------------------------- floor --

def pairs(c):
    """Query-key pairs of one head and batch row that the masks leave (key padding leaves half of them on average)."""
    n = c["Tq"] * (c["Tq"] + 1) / 2 if c["causal"] else c["Tq"] * c["Tk"]
    return n / 2 if c["masked"] else n


def work(case):
    c = case
    if c["kind"] == "attn":
        e, C = 2 if c["type"] == "f16" else 4, c["heads"] * c["hd"]
        # q, o, do, dq and k, v, dk, dv; five products: scores, dp, dq, dk, dv
        return {"bytes": 4.0 * e * c["batch"] * C * (c["Tq"] + c["Tk"]), "flops": 10.0 * c["batch"] * C * pairs(c)}
    if c["kind"] == "norm":
        n, e = c["rows"] * c["d"], 2 if c["type"] == "f16" else 4
        return {"bytes": n * (8.0 + e + (4 if c["residual"] else 0)) + (12.0 * c["d"] if c["affine"] else 0), "flops": 15.0 * n}
    if c["kind"] == "geglu":
        n, e = c["rows"] * c["F"], 2 if c["type"] == "f16" else 4
        return {"bytes": n * (8.0 + 3 * e), "flops": 30.0 * n}
    if c["kind"] == "geglu_gemm":
        M, F, K = c["M"], c["F"], c["K"]
        return {"bytes": 2.0 * M * K + 2 * F * K * 34 / 32 + (8 * F if c["bias"] else 0) + 6.0 * M * F, "flops": 4.0 * M * F * K}
    M, N, K, e = c["M"], c["N"], c["K"], 2 if c["type"] == "f16" else 4
    return {"bytes": e * M * (N + K) + N * K * 34 / 32, "flops": 2.0 * M * N * K}


# ----------------------------------------------------------- 64-bit result --

def weight64(raw, n, k):
    b = raw.reshape(n * (k // 32), 34)
    q = b[:, 2:].contiguous().view(torch.int8).double()
    return (q * b[:, :2].contiguous().view(torch.float16).double()).view(n, k)


def attn_exact(c, s):
    """One head of one batch row at a time, over the keys that its length leaves: P = softmax(S), dS = P (dP - sum P dP)."""
    grads = [torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) for n in ("q", "k", "v")]
    scale = c["hd"] ** -0.5
    for b in range(c["batch"]):
        L = c["Tk"] if s["lens"] is None else int(s["lens"][b])
        for h in range(c["heads"]):
            col = slice(h * c["hd"], (h + 1) * c["hd"])
            q, do = s["q"][b, :, col].double(), s["do"][b, :, col].double()
            k, v = s["k"][b, :L, col].double(), s["v"][b, :L, col].double()
            sc = torch.mm(q, k.t().contiguous()) * scale
            if c["causal"]:
                sc.masked_fill_(torch.ones(c["Tq"], L, dtype=torch.bool, device=DEV).triu(1), -math.inf)
            p = torch.softmax(sc, 1)
            dp = torch.mm(do, v.t().contiguous())
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            grads[0][b, :, col] = torch.mm(ds, k)
            grads[1][b, :L, col] = torch.mm(ds.t().contiguous(), q)
            grads[2][b, :L, col] = torch.mm(p.t().contiguous(), do)
    return grads


def norm_exact(c, s):
    x, dy = s["x"].double(), s["dy"].double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    r = (var + 1e-5).rsqrt()
    n = (x - mean) * r
    w = dy * s["gamma"].double() if s["gamma"] is not None else dy
    dx = (w - (w.sum(1, keepdim=True) + n * (w * n).sum(1, keepdim=True)) / c["d"]) * r
    if s["res"] is not None:
        dx += s["res"].double()
    return [dx] + ([torch.einsum("rd,rd->d", dy, n), dy.sum(0)] if c["affine"] else [])


def gate64(v, g, dy):
    cdf = torch.special.ndtr(g)
    pdf = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return torch.cat([dy * g * cdf, dy * v * (cdf + g * pdf)], 1)


def exact(case, seed):
    c = case
    s = INPUTS[c["kind"]](c, seed)
    if c["kind"] == "attn":
        return attn_exact(c, s)
    if c["kind"] == "norm":
        return norm_exact(c, s)
    if c["kind"] == "geglu":
        h = s["h"].double()
        return [gate64(h[:, :c["F"]], h[:, c["F"]:], s["dy"].double())]
    if c["kind"] == "geglu_gemm":
        h = torch.mm(s["A"].double(), weight64(s["W"], 2 * c["F"], c["K"]).t().contiguous())
        if s["bias"] is not None:
            h += s["bias"].double()
        return [gate64(h[:, :c["F"]], h[:, c["F"]:], s["dG"].double())]
    return [torch.mm(s["dC"].double(), weight64(s["W"], c["N"], c["K"]))]
