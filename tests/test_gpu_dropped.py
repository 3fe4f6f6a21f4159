"""Tokens and rows that have no place are told."""
import numpy as np
import pytest

import _decode as D
from test_gpu_attend import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("entry", [-1, 2**31 - 1])
def test_a_new_token_without_a_page(vs, dtype, entry):
    c = Case(vs, [40, 64, 0], 4, 2, 32, 32, dtype)
    c.table[1, 1] = entry
    c.sequences(np.zeros(c.cache.npages, np.int32))
    A = vs.DeviceArray
    kb, k = D.stored(c.rng.standard_normal((3, 2, 32)), dtype)
    out = A((3, 4, 32), dtype)
    c.cache.attend(c.seqs, A.of(c.qb, dtype), out, k=A.of(kb, dtype), v=A.of(kb, dtype))
    with pytest.raises(ValueError, match="no page"):
        c.cache.check()
    c.cache.check()
    D.write_rows(c.pool[:, 0], c.table, 0, 39, kb[:1], kb[:1], 32, dtype)  # the one that has a place is stored
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))
    c.k[0][-1] = c.v[0][-1] = k[0]
    got = D.from_bf16(out.numpy()) if dtype == "bf16" else out.numpy()
    for b, seen in ((0, np.arange(40)), (1, np.arange(32)), (2, np.arange(0))):
        args = (c.q[b], c.k[b], c.v[b], seen, 32 ** -0.5)
        D.assert_rounded(got[b], D.attend(*args)[0], D.attend_tolerance(*args, dtype)[0], dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_appended_rows_past_the_table(vs, dtype, rows):
    """Those that have a column are stored, the others told."""
    c = Case(vs, [96, 60], 2, 2, 48, 32, dtype, width=3)
    lens = np.array([98, 60], np.int32)  # two positions past the first one's columns
    A = vs.DeviceArray
    seqs = vs.KVSequences(A.of(c.table, "i32"), A.of(lens, "i32"), A.of(np.zeros(c.cache.npages), "i32"))
    kb, _ = D.stored(c.rng.standard_normal((rows + 3, 2, 48)), dtype)
    vb, _ = D.stored(c.rng.standard_normal((rows + 3, 2, 48)), dtype)
    c.cache.append(seqs, A.of(kb, dtype), A.of(vb, dtype), starts=A.of([0, rows, rows + 3], "i32"))
    with pytest.raises(ValueError, match="outgrew"):
        c.cache.check()
    for b, r0, n in ((0, 0, rows), (1, rows, 3)):
        for j in range(n):
            if lens[b] - n + j < 96:
                D.write_rows(c.pool[:, 0], c.table, b, lens[b] - n + j, kb[r0 + j:r0 + j + 1], vb[r0 + j:r0 + j + 1], 32, dtype)
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))
    c.cache.check()
