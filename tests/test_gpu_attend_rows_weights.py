"""How exactly attention of a few rows per sequence holds the softmax's weights: answers of bf16 caches are those of
32-bit weights, rounded once, as those of one new token are."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,rows,dim", [(7, 5, 128), (40, 5, 64), (40, 1, 16), (3000, 5, 128), (3000, 1, 96), (500, 4, 256)])
def test_weights_of_few_rows_are_held_in_32_bits(vs, dtype, causal, n, rows, dim):
    """Two positions that count, the first two, of values 0 and v at scores 0 and -a: the answer is v w / (1 + w),
    w = exp(-a).  All others are at -200 and below, whose weights are 0 in 32 bits (and 1e-87 in truth).

    a <= 8 is exact, and so is its product.  In 32 bits: scale * log2(e) and its product are off by 2^-24 of the
    exponent each, which is 8 * 2^-23 = 2^-20 of w at most; exp2 by 2^-22; the sum, the quotient, the product with it
    and the factors of a join by less than 2^-21 together; three parts of a weight are added up by units that may
    truncate, 3 * 2^-23.  Below 2^-18 of the answer, then the last rounding.  (A weight rounded to bf16 is off by up to
    2^-8.)  Rows times heads of a group: 12 to 60, at most 64 per sequence."""
    rng = np.random.default_rng(n + dim)
    A, kv, group, nseq = vs.DeviceArray, 4, 12, 3
    heads, width = kv * group, -(-n // 32) + 1
    k, v = np.zeros((nseq * n, kv, dim)), np.zeros((nseq * n, kv, dim))
    k[..., 1], v[...] = -200, 1
    k[::n], v[::n] = 0, 0
    k[1::n, :, :2] = [-1, 0]
    v[1::n] = rng.standard_normal((nseq, kv, dim))
    q = np.zeros((nseq * rows, heads, dim))
    q[..., 0] = np.exp(rng.uniform(np.log(0.01), np.log(8), q.shape[:2]))
    q[..., 1] = 1
    (kb, k), (vb, v), (qb, q) = (D.stored(x, dtype) for x in (k, v, q))
    cache = vs.PagedKVCache(nseq * width, 32, kv, dim, dtype=dtype)
    seqs = cache.new_sequences(nseq, width)
    cache.extend(seqs, n)
    cache.append(seqs, A.of(kb, dtype), A.of(vb, dtype), starts=A.of(n * np.arange(nseq + 1), "i32"))
    out = A(q.shape, dtype)
    cache.attend_rows(seqs, A.of(qb, dtype), out, starts=A.of(rows * np.arange(nseq + 1), "i32"), scale=1.0, causal=causal)
    cache.check()
    w = np.exp(-q[..., 0].astype(np.float64)).reshape(nseq, rows, kv, group, 1)
    exact = (w / (1 + w) * v[1::n].astype(np.float64)[:, None, :, None]).reshape(q.shape)
    got = D.from_bf16(out.numpy()) if dtype == "bf16" else out.numpy()
    D.assert_rounded(got, exact, 2.0 ** -18 * np.abs(exact), dtype)
    cache.close()
