"""How exactly rotary positions hold their angles: small ones, and those of frequencies of very many turns."""
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TURN = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def angle(w, p):
    """w p less whole turns, in radians (w a double; exact but for the last rounding)."""
    t = Fraction(float(w)) * p / TURN
    return float((t - round(t)) * TURN)


def cos_sin(vs, w, positions):
    """What (1, 0) becomes: cosines and sines [positions, pairs]."""
    A, n = vs.DeviceArray, len(w)
    rot = vs.Rotary(2 * n, frequencies=w)
    x = np.zeros((len(positions), 1, 2 * n), np.float32)
    x[..., :n] = 1
    out = A(x.shape, "f32")
    rot.rotate(A.of(x, "f32"), out, A.of(positions, "i32"))
    rot.close()
    y = out.numpy()[:, 0].astype(np.float64)
    return y[:, :n], y[:, n:]


def test_small_angles(vs):
    """Slow pairs at early positions: angles about 2^-32 of a turn and below it are not cut off.

    The angle is off by 2^-64 of a turn per position (below 2^-25 of any here), by its words' and factors' roundings to
    fp32 (5 of 2^-24 of it at most: two conversions, a factor each, a product, a sum); sin x = x (1 - x^2 / 6) by two more,
    the gain's product and the pair's by one each: below 2^-20 of the sine in all."""
    w = np.concatenate([2 * np.pi * 2.0 ** -32 * np.array([0.01, 0.3, 0.9, 0.999, 1.0, 1.5, 3.9, -0.5, -1.7, 40.3]),
                        10000.0 ** -np.arange(2, 2.5, 0.1)])
    pos = np.array([1, 2, 3, 7, -1, -5])
    _, s = cos_sin(vs, w, pos)
    want = np.array([[np.sin(angle(wi, int(p))) for wi in w] for p in pos])
    np.testing.assert_allclose(s, want, rtol=2.0 ** -20, atol=0)


def test_frequencies_of_many_turns(vs):
    """Up to 2^40 radians per position, at positions up to 2^31: within 2^-33 of a turn (7.4e-10 radians), 2^-22 of the
    angle (up to pi / 4) as above, what the polynomials leave out (1.8e-9) and their and the products' roundings (4 of
    2^-24): below 6e-7 in all."""
    rng = np.random.default_rng(0)
    w = np.concatenate([2.0 ** np.arange(0, 40, 3.0) * (1 + rng.random(14)), [2.0 ** 40, -(2.0 ** 40), 1e12 / 3, 0.1, 7.0]])
    pos = np.concatenate([[1, 2**31 - 1, -2**31], rng.integers(-2**31, 2**31, 40)])
    c, s = cos_sin(vs, w, pos)
    x = np.array([[angle(wi, int(p)) for wi in w] for p in pos])
    np.testing.assert_allclose(c, np.cos(x), rtol=0, atol=6e-7)
    np.testing.assert_allclose(s, np.sin(x), rtol=0, atol=6e-7)
