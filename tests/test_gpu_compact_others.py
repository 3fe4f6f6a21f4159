"""Compaction beside other holders of pages: their tables follow, and a map tells where pages went."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu


class Two:
    """Two sets of sequences on one set of counts, a page that both share, one held by the caller alone."""

    def __init__(self, vs, npages, dtype="bf16"):
        self.vs, A = vs, vs.DeviceArray
        rng = np.random.default_rng(npages)
        ids = rng.permutation(npages)
        self.first = np.array([[ids[0], ids[1], -1], [ids[2], -1, ids[3]]], np.int32)
        self.second = np.array([[ids[4], ids[0]], [npages, ids[5]], [-1, -7]], np.int32)
        self.hold = int(ids[6])
        refs = np.zeros(npages, np.int32)
        np.add.at(refs, np.concatenate([self.first[self.first >= 0], ids[[4, 0, 5, 6]]]), 1)
        self.model = D.Pages(self.first, [60, 90], refs, 32)
        self.pool, _ = D.stored(rng.standard_normal((npages, 1, 2, 2, 32 * 16)), dtype)
        self.mem = A.of(self.pool, dtype)
        self.cache = vs.PagedKVCache(npages, 32, 2, 16, dtype=dtype, memory=self.mem)
        self.refs = A.of(refs, "i32")
        self.a = vs.KVSequences(A.of(self.first, "i32"), A.of([60, 90], "i32"), self.refs)
        self.b = vs.KVSequences(A.of(self.second, "i32"), A.of([40, 64, 0], "i32"), self.refs)
        self.moved = A.of(np.full(npages, 99), "i32")


@pytest.mark.parametrize("npages", [8, 300, 16384, 16385, 40_000])
@pytest.mark.parametrize("apart", [False, True])
def test_other_tables_follow(vs, npages, apart):
    t = Two(vs, npages)
    out = t.a
    if apart:
        A = vs.DeviceArray
        out = vs.KVSequences(A.of(np.full((2, 3), 9), "i32"), A.of([9, 9], "i32"), t.refs)
    t.cache.compact(t.a, out, others=[t.b], moved=t.moved)
    t.cache.check()
    want = t.model.compact()
    where = np.arange(npages)
    for src, to in want.copies:
        where[src] = to
    assert np.array_equal(out.table.numpy(), want.table) and np.array_equal(t.refs.numpy(), want.refs)
    valid = (t.second >= 0) & (t.second < npages)
    assert np.array_equal(t.b.table.numpy(), np.where(valid, where[np.where(valid, t.second, 0)], t.second))
    assert t.b.lens.numpy().tolist() == [40, 64, 0]
    assert np.array_equal(t.moved.numpy(), where)
    # what every holder names holds what it held
    pool = t.mem.numpy()
    for before, after in ((t.first, out.table.numpy()), (t.second, t.b.table.numpy()), ([t.hold], [where[t.hold]])):
        for p, q in zip(np.ravel(before), np.ravel(after)):
            if 0 <= p < npages:
                assert np.array_equal(pool[q], t.pool[p])


def test_a_map_alone(vs):
    t = Two(vs, 50)
    t.cache.compact(t.a, others=[t.b])
    t.cache.compact(t.a, moved=t.moved, others=[t.b])  # nothing is left to move
    assert np.array_equal(t.moved.numpy(), np.arange(50))


def test_refusals(vs):
    t, A = Two(vs, 20), vs.DeviceArray
    elsewhere = vs.KVSequences(t.b.table, t.b.lens, A.of(np.zeros(20), "i32"))
    for bad in (dict(others=[elsewhere]), dict(others=[t.a]), dict(others=[t.b, t.b]),
                dict(out=vs.KVSequences(A((2, 3), "i32"), A((2,), "i32"), A((20,), "i32")), others=[t.b]),
                dict(moved=A((19,), "i32")), dict(moved=A((20,), "f32")),
                dict(others=[vs.KVSequences(t.b.table, t.b.lens, A((21,), "i32"))])):
        with pytest.raises(ValueError):
            t.cache.compact(t.a, **bad)
    t.cache.check()
    assert np.array_equal(t.a.table.numpy(), t.first) and np.array_equal(t.mem.numpy(), t.pool)
