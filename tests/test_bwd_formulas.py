"""The 64-bit formulas that the backward operators are tested against, against central differences of the forward pass.

With eps = 2^-10 and values of order 1 the third derivative's share is under 2^-18 of a gradient's scale, the differences'
rounding under 2^-40."""
import numpy as np
import pytest

import bwd_block
import bwd_ref

EPS, TOL = 2.0 ** -10, 2.0 ** -17


def differences(f, x):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        for s in (1, -1):
            y = x.copy()
            y[i] += s * EPS
            g[i] += s * f(y) / (2 * EPS)
    return g


def close(got, want):
    assert np.all(np.abs(got - want) <= TOL * max(1.0, np.abs(want).max())), np.abs(got - want).max()


@pytest.mark.parametrize("causal,keys", [(False, 5), (True, 5), (True, 2), (False, 0)])
def test_attention(causal, keys):
    r = bwd_ref.rng_of(1)
    q, k, v, do = (r.standard_normal((n, 3)) for n in (6, 5, 5, 6))
    i, j = np.arange(6)[:, None], np.arange(5)[None, :]
    seen, sc = (j < keys) & ((j <= i) | (not causal)), 0.7

    def out(q, k, v):
        return bwd_ref.softmax_rows(np.where(seen, q @ k.T * sc, -np.inf)) @ v

    want, _ = bwd_ref.attn_head(q, k, v, do, sc, seen, "f32", out(q, k, v))
    close(want[0], differences(lambda x: (out(x, k, v) * do).sum(), q))
    close(want[1], differences(lambda x: (out(q, x, v) * do).sum(), k))
    close(want[2], differences(lambda x: (out(q, k, x) * do).sum(), v))
    if keys == 0:
        assert not any(np.any(w) for w in want)


def test_geglu():
    r = bwd_ref.rng_of(2)
    v, g, dy = r.standard_normal((3, 4, 7)) * 1.5
    want = bwd_ref.geglu_parts(v, g, dy)
    close(want[0], differences(lambda x: (x * bwd_block.gelu(g) * dy).sum(), v))
    close(want[1], differences(lambda x: (v * bwd_block.gelu(x) * dy).sum(), g))


def test_norm():
    r = bwd_ref.rng_of(3)
    x, dy = r.standard_normal((2, 4, 9))
    gm, bt = r.standard_normal((2, 9))
    want = bwd_block.norm_bwd(x, gm, dy)
    close(want[0], differences(lambda t: (bwd_block.norm_fwd(t, gm, bt) * dy).sum(), x))
    close(want[1], differences(lambda t: (bwd_block.norm_fwd(x, t, bt) * dy).sum(), gm))
    close(want[2], differences(lambda t: (bwd_block.norm_fwd(x, gm, t) * dy).sum(), bt))


def test_block():
    blk = bwd_block.Block()
    s = blk.forward(blk.x, blk.ctx)
    bwd_block.check_differences(blk, blk.backward(s, bwd_ref.f64(blk.dy)), 0.0)
