"""The 64-bit gradients that the GroupNorm tests hold the kernels to, against differences of the 64-bit forward pass."""
import numpy as np
import pytest

import norm_i8_ref as ref


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("B,P,C,G", [(1, 1, 8, 2), (2, 7, 12, 3), (1, 20, 5, 1)])
def test_gradients_against_differences(B, P, C, G, act):
    rng = ref.rng_of(7)
    x = rng.standard_normal((B, P, C)) * 1.5 + 0.3
    gamma, beta, dy = 1 + 0.2 * rng.standard_normal(C), 0.3 * rng.standard_normal(C), rng.standard_normal((B, P, C))

    def f(x, gamma, beta):
        return float((ref.forward64(ref.Group(x, G, 1e-3), gamma, beta, act, x.shape)[0] * dy).sum())

    (dx, _), (dg, _), (db, _) = ref.backward64(ref.Group(x, G, 1e-3), dy, gamma, beta, act, None)
    size = np.sqrt((dx ** 2).sum() + (dg ** 2).sum() + (db ** 2).sum())
    for _ in range(4):
        d = [rng.standard_normal(t.shape) for t in (x, gamma, beta)]
        n = np.sqrt(sum((t ** 2).sum() for t in d))
        d = [t / n for t in d]
        e = 1e-4
        want = (f(x + e * d[0], gamma + e * d[1], beta + e * d[2]) - f(x - e * d[0], gamma - e * d[1], beta - e * d[2])) / (2 * e)
        have = (dx * d[0]).sum() + (dg * d[1]).sum() + (db * d[2]).sum()
        # central differences: e^2 times the third derivative (eps 1e-3 lets inv grow to 30 where a group has few values), and 1e-16 / e
        assert abs(have - want) <= 1e-5 * max(size, 1.0), (have, want)


def test_codes_by_definition():
    x = np.array([[127.0, 0.5, 1.5, -2.5, 126.5], [0.0, 0, 0, 0, 0], [1.0, np.inf, 0, 0, 0], [np.nan, 1, 2, 3, 4]], np.float32)
    q, s = ref.codes_of(x)
    assert q.tolist() == [[127, 0, 2, -2, 126], [0] * 5, [0] * 5, [0] * 5]
    assert s[0] == 1 and s[1] == np.float32(2.0 ** -126) and np.isnan(s[2:]).all()
