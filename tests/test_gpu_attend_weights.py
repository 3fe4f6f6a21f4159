"""How exactly attention holds the softmax's weights: answers of bf16 caches are
those of 32-bit weights, rounded once."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 33, 3000])
def test_weights_are_held_in_32_bits(vs, dtype, n):
    """Two positions that count, of values 0 and v, at scores 0 and -a: the answer is v w / (1 + w), w = exp(-a).
    All others are at -200 and below, whose weights are 0 in 32 bits (and 1e-87 in truth).

    a <= 8 is exact, and so is its product.  In 32 bits: scale * log2(e) and its product are off by 2^-24 of the
    exponent each, which is 8 * 2^-23 = 2^-20 of w at most; exp2 by 2^-22; the sum, the reciprocal (2^-23), the product
    with it and the factors of up to two joins (2^-22 in all) by less than 2^-21 together.  Below 2^-19 of the answer,
    then the last rounding.  (Weights of 16 bits are off by up to 2^-17, and a few of these 8,192 answers round to
    the other neighbour.)"""
    rng = np.random.default_rng(n)
    A, heads, dim = vs.DeviceArray, 64, 128
    width = -(-n // 32) + 1
    k, v = np.zeros((n, 1, dim)), np.zeros((n, 1, dim))
    k[1:, 0, 1] = -200
    k[-1, 0, :2] = [-1, 0]
    v[-1] = rng.standard_normal((1, dim))
    v[1:-1] = 1
    q = np.zeros((1, heads, dim))
    q[0, :, 0] = np.exp(rng.uniform(np.log(0.01), np.log(8), heads))
    q[0, :, 1] = 1
    (kb, k), (vb, v), (qb, q) = (D.stored(x, dtype) for x in (k, v, q))
    cache = vs.PagedKVCache(width, 32, 1, dim, dtype=dtype)
    seqs = cache.new_sequences(1, width)
    cache.extend(seqs, n)
    cache.append(seqs, A.of(kb, dtype), A.of(vb, dtype), starts=A.of([0, n], "i32"))
    out = A((1, heads, dim), dtype)
    cache.attend(seqs, A.of(qb, dtype), out, scale=1.0)
    cache.check()
    w = np.exp(-q[0, :, 0].astype(np.float64))[:, None]
    exact = w / (1 + w) * v[-1].astype(np.float64)
    got = D.from_bf16(out.numpy()) if dtype == "bf16" else out.numpy()
    D.assert_rounded(got[0], exact, 2.0 ** -19 * np.abs(exact), dtype)
    cache.close()
