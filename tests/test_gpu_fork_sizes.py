"""Forks of every size around where one workgroup stops doing them, against the model."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("npages,n,nout,width", [(4000, 20, 20, 40), (4100, 20, 30, 40), (4093, 25, 25, 40), (4094, 25, 25, 40),
                                                 (100, 700, 900, 2), (100, 1024, 1024, 1), (100, 1025, 3, 1), (30, 3, 1025, 1),
                                                 (6000, 4, 4, 17), (6000, 4, 4, 18), (1, 1, 1, 0), (5, 2, 0, 3), (20_000, 300, 200, 30)])
@pytest.mark.parametrize("same_counts", [False, True])
def test_forks(vs, npages, n, nout, width, same_counts):
    A, rng = vs.DeviceArray, np.random.default_rng(npages + n)
    cache = vs.PagedKVCache(npages, 32, 1, 16)
    table = rng.integers(-1, npages + 1, (n, width)).astype(np.int32)  # (entries that are no page among them)
    lens = rng.integers(0, 32 * width + 1, n).astype(np.int32)
    valid = (table >= 0) & (table < npages)
    refs = np.bincount(table[valid], minlength=npages).astype(np.int32)
    parents = rng.integers(-1, n, nout).astype(np.int32)
    m = D.Pages(np.where(valid, table, -1), lens, refs, 32).fork(parents)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of(lens, "i32"), A.of(refs, "i32"))
    out = vs.KVSequences(A.of(np.full((nout, width), 77), "i32"), A.of(np.full(nout, 77), "i32"),
                         seqs.refs if same_counts else A.of(np.full(npages, 77), "i32"))
    cache.fork(seqs, A.of(parents, "i32"), out)
    cache.check()
    want = np.where((parents >= 0)[:, None], table[np.where(parents >= 0, parents, 0)], -1)
    assert np.array_equal(out.table.numpy(), want) and np.array_equal(out.lens.numpy(), m.lens)
    assert np.array_equal(out.refs.numpy(), m.refs)
    if not same_counts:
        assert np.array_equal(seqs.refs.numpy(), refs)
    assert np.array_equal(seqs.table.numpy(), table)
    cache.close()
