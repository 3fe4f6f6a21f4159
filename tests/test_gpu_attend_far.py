"""Attention of many rows at the last positions that there can be."""
import numpy as np
import pytest

import _decode as D
import _prompt as P
from test_gpu_attend_tiles import kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,tile,rows", [(512, (256, False), 256), (1, (64, True), 5)])
@pytest.mark.parametrize("missing", [False, True])
def test_last_positions(vs, kv, tile, rows, missing):
    """A length of 2^31 - 32 behind a window, an even and an odd number of blocks: what fills an odd step up is no
    position of the sequence's."""
    A, rng, dim, window = vs.DeviceArray, np.random.default_rng(kv), 16, 100
    width = (2**31 - 1) // 32
    n, held = width * 32, 14
    assert kernel(vs, rows, kv, kv, 1, width, 32, dim, "bf16") == tile
    table = np.full((1, width), -1, np.int32)
    table[0, -held:] = rng.permutation(held)
    if missing:
        table[0, -6] = -1
    seqs = vs.KVSequences(A.of(table, "i32"), A.of([n], "i32"), A.of(np.zeros(held), "i32"))
    cache = vs.PagedKVCache(held, 32, kv, dim)
    last = np.arange(held * 32 - rows, held * 32)  # (of the positions that are held)
    seen = P.seen_mask(last, held * 32, window, 0)
    if missing:
        seen[:, (held - 6) * 32:(held - 5) * 32] = False
    (kb, k), (vb, v) = (D.stored(rng.standard_normal((held * 32, 1, dim)), "bf16") for _ in range(2))
    qb, q = D.stored(2 * rng.standard_normal((rows, 1, dim)), "bf16")
    wide = lambda x: A.of(np.repeat(x, kv, 1), "bf16")  # noqa: E731
    cache.append(seqs, wide(kb), wide(vb), starts=A.of([0, held * 32], "i32"))
    out, lse = A((rows, kv, dim), "bf16"), A((rows, kv), "f32")
    cache.attend_rows(seqs, wide(qb), out, lse=lse, starts=A.of([0, rows], "i32"), window=window)
    cache.check()
    got, got_lse = D.from_bf16(out.numpy()), lse.numpy()
    assert (got == got[:, :1]).all() and (got_lse == got_lse[:, :1]).all()
    eo, el, to, tl = P.attend_rows(*(x.astype(np.float64) for x in (q, k, v)), seen, dim ** -0.5, "bf16")
    D.assert_rounded(got[:, :1], eo, to, "bf16")
    assert (np.abs(got_lse[:, :1] - el) <= tl).all()
    cache.close()


def test_as_many_sequences_as_there_may_be(vs):
    """2^20 of them, one row each, 8 key-value heads: 8.5 million workgroups of 256 threads are a launch that the runtime
    takes (below 2^32 threads).  Each sees one position of a page that it has to itself or shares."""
    A, rng, n, kv, dim, held = vs.DeviceArray, np.random.default_rng(3), 2**20, 8, 16, 64
    table = rng.integers(0, held, (n, 1)).astype(np.int32)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of(np.ones(n), "i32"), A.of(np.zeros(held), "i32"))
    cache = vs.PagedKVCache(held, 32, kv, dim)
    own = vs.KVSequences(A.of(np.arange(held)[:, None], "i32"), A.of(np.ones(held), "i32"), seqs.refs)
    kb, vb = (D.stored(rng.standard_normal((held, kv, dim)), "bf16")[0] for _ in range(2))
    cache.append(own, A.of(kb, "bf16"), A.of(vb, "bf16"))
    q, out = A.of(np.full((n, kv, dim), 0x3F80), "bf16"), A((n, kv, dim), "bf16")
    cache.attend_rows(seqs, q, out)
    cache.check()
    assert np.array_equal(out.numpy(), vb[table[:, 0]])  # a single weight: the value itself
    cache.close()
