"""The cache's pages against their rules: extending with copies on write,
forking, freeing, evicting, compacting, copying."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu


class Pool:
    """A cache whose every page holds its own number pattern, and sequences on it."""

    def __init__(self, vs, npages, table, lens, page=32, layers=2, kv=2, dim=16, dtype="bf16", held=None):
        self.vs, self.page, self.npages = vs, page, npages
        rng = np.random.default_rng(1)
        shape = (npages, layers, 2, kv, page * dim)
        self.pool = (rng.integers(0, 1 << 16, shape).astype(np.uint16) if dtype == "bf16"
                     else rng.standard_normal(shape).astype(np.float32))
        self.mem = vs.DeviceArray.of(self.pool, dtype)
        self.cache = vs.PagedKVCache(npages, page, kv, dim, layers=layers, dtype=dtype, memory=self.mem)
        table, lens = np.array(table, np.int32), np.array(lens, np.int32)
        refs = np.bincount(table[table >= 0], minlength=npages).astype(np.int32)
        if held is not None:  # pages that someone else holds too
            np.add.at(refs, held, 1)
        self.model = D.Pages(table, lens, refs, page)
        self.seqs = self.put(self.model)

    def put(self, m):
        A = self.vs.DeviceArray
        return self.vs.KVSequences(A.of(m.table, "i32"), A.of(m.lens, "i32"), A.of(m.refs, "i32"))

    def spare(self, n):
        A = self.vs.DeviceArray
        w = self.model.table.shape[1]
        return self.vs.KVSequences(A.of(np.full((n, w), 99), "i32"), A.of(np.full(n, 99), "i32"),
                                   A.of(np.full(self.npages, 99), "i32"))

    def agrees(self, seqs=None):
        s, m = seqs or self.seqs, self.model
        assert np.array_equal(s.table.numpy(), m.table)
        assert np.array_equal(s.lens.numpy(), m.lens)
        assert np.array_equal(s.refs.numpy(), m.refs)
        for a, b in m.copies:
            self.pool[b] = self.pool[a]
        m.copies = []
        assert np.array_equal(self.mem.numpy().view(np.uint16), self.pool.view(np.uint16))

    def extend(self, counts, seqs=None):
        A = self.vs.DeviceArray
        n = len(self.model.lens)
        self.cache.extend(seqs or self.seqs, counts if isinstance(counts, int) else A.of(np.array(counts), "i32"))
        return self.model.extend(np.full(n, counts) if isinstance(counts, int) else np.array(counts))

    def fork(self, parents, seqs=None):
        out = self.spare(len(parents))
        self.cache.fork(seqs or self.seqs, self.vs.DeviceArray.of(np.array(parents), "i32"), out)
        self.model = self.model.fork(parents)
        self.seqs = out


def rows(width, *seqs):
    return [list(s) + [-1] * (width - len(s)) for s in seqs]


@pytest.mark.parametrize("dtype,layers,kv,dim", [("bf16", 1, 1, 16), ("f32", 3, 2, 48), ("bf16", 2, 5, 80)])
def test_extend_takes_the_lowest_free_pages(vs, dtype, layers, kv, dim):
    p = Pool(vs, 20, rows(5, [7, 2], [9], [], [4, 0, 1]), [64, 5, 0, 96], layers=layers, kv=kv, dim=dim, dtype=dtype)
    for c in (1, 31, 1, [0, 40, -3, 2]):
        assert p.extend(c) is None
        p.cache.check()
        p.agrees()


def test_extend_copies_shared_last_pages(vs):
    """Shared by two that go on (the first keeps it); by one that goes on and one that does not; held from outside;
    shared but full; shared by three."""
    table = rows(3, [0, 1], [0, 1], [2], [2], [3], [4], [4], [5], [5], [5])
    lens = [40, 40, 10, 10, 7, 32, 32, 1, 1, 1]
    for counts in (1, [1, 1, 0, 1, 1, 1, 1, 1, 1, 1], [1, 0, 0, 0, 0, 0, 1, 0, 1, 1], [30] * 10):
        p = Pool(vs, 24, table, lens, held=[3])
        assert p.extend(counts) is None
        p.cache.check()
        p.agrees()


def test_extend_refuses_whole(vs):
    """Too few pages, or a table row too short: nothing changes and check() tells."""
    p = Pool(vs, 6, rows(4, [0, 1], [2], [3]), [64, 5, 6])
    assert p.extend([100, 0, 0]) == "width"
    with pytest.raises(ValueError, match="table row"):
        p.cache.check()
    p.agrees()
    assert p.extend([33, 28, 28]) == "pages"  # four wanted, two free
    with pytest.raises(vs.VsError, match="2 pages short"):
        p.cache.check()
    p.agrees()
    p.cache.check()  # told once
    assert p.extend([32, 28, 0]) is None
    p.cache.check()
    p.agrees()


def test_fork_and_free(vs):
    p = Pool(vs, 16, rows(4, [0, 1, 2], [0, 1, 3], [4], [], [5, -1, 6]), [70, 80, 9, 0, 90], held=[4, 15])
    p.fork([1, 1, -1, 3, 0, 1, 4])
    p.cache.check()
    p.agrees()
    p.fork([0, 5, 6, 4])
    p.agrees()
    A = vs.DeviceArray
    p.cache.free(p.seqs, A.of([1, 1, 99, -1], "i32"))
    for b in [1]:
        np.subtract.at(p.model.refs, p.model.table[b][p.model.table[b] >= 0], 1)
        p.model.table[b], p.model.lens[b] = -1, 0
    p.agrees()
    p.cache.free(p.seqs)
    p.model = D.Pages(np.full_like(p.model.table, -1), 0 * p.model.lens, p.model.refs, 32)
    p.model.refs[:] = 0
    p.model.refs[[4, 15]] = 1  # someone else's
    p.agrees()


def test_fork_reports_bad_parents(vs):
    p = Pool(vs, 8, rows(2, [0], [1]), [3, 4])
    out = p.spare(3)
    p.cache.fork(p.seqs, vs.DeviceArray.of([0, 2, -2], "i32"), out)
    with pytest.raises(ValueError, match="parent"):
        p.cache.check()
    p.model = p.model.fork([0, -1, -1])
    p.agrees(out)


def test_fork_in_one_set_of_counts(vs):
    """refs may be one buffer for both sides."""
    p = Pool(vs, 8, rows(3, [0, 1], [0, 2]), [50, 60])
    A = vs.DeviceArray
    out = vs.KVSequences(A.of(np.zeros((4, 3)), "i32"), A.of(np.zeros(4), "i32"), p.seqs.refs)
    p.cache.fork(p.seqs, A.of([[1, 1], [1, 0]], "i32"), out)
    p.model = p.model.fork([1, 1, 1, 0])
    p.agrees(out)


@pytest.mark.parametrize("npages,live", [(10, 4), (4096, 1000), (4097, 4000), (9000, 3), (5, 5), (70, 0), (16384, 8192),
                                         (16385, 8000), (20_001, 15_000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(vs, npages, live, in_place):
    rng = np.random.default_rng(npages)
    ids = rng.permutation(npages)[:live]
    width = max(1, -(-live // 3)) + 1
    table = np.full((4, width), -1, np.int32)
    for i, part in enumerate(np.array_split(ids, 3)):
        table[i, :len(part)] = part
    table[3] = table[0]
    if live > 3:
        table[1, 1] = -1
    p = Pool(vs, npages, table, [32 * width - 3] * 4, layers=1, kv=1, held=ids[-1:] if live else None)
    out = p.seqs if in_place else p.spare(4)
    p.cache.compact(p.seqs, None if in_place else out)
    p.cache.check()
    p.model = p.model.compact()
    p.agrees(out)
    n = int((p.model.refs > 0).sum())
    assert (out.refs.numpy()[:n] > 0).all() and not out.refs.numpy()[n:].any()


def test_evict_frees_what_no_window_sees(vs):
    table = rows(6, [0, 1, 2, 3, 4, 5], [0, 6, 7], [8])
    p = Pool(vs, 10, table, [190, 96, 4])
    p.cache.evict(p.seqs, 50, 33)
    p.cache.check()
    # sequence 0: positions 33 .. 139 are out of sight: pages 2 and 3; sequence 1: 33 .. 45, no whole page
    p.model.table[0, [2, 3]] = -1
    p.model.refs[[2, 3]] -= 1
    p.agrees()
    p.cache.evict(p.seqs, 1, 0)
    p.model.table[0, [0, 1, 4]] = -1
    p.model.table[1, [0, 1]] = -1
    p.model.refs[[0, 0, 1, 4, 6]] -= 1
    p.model.refs[0] = 0
    p.agrees()


@pytest.mark.parametrize("layers,kv,dim", [(1, 1, 16), (1, 3, 240), (5, 2, 128)])
def test_copy_pages(vs, layers, kv, dim):
    p = Pool(vs, 9, rows(1, [0]), [1], layers=layers, kv=kv, dim=dim)
    A = vs.DeviceArray
    p.cache.copy(A.of([0, 3, 3, 9, 4], "i32"), A.of([8, 7, 6, 5, -1], "i32"))
    p.cache.check()
    p.pool[8], p.pool[7], p.pool[6] = p.pool[0], p.pool[3], p.pool[3]
    p.agrees()


@pytest.mark.parametrize("n", [1500, 1024, 700])
def test_many_sequences_and_pages(vs, n):
    """Up to and past one workgroup's threads, with most last pages shared."""
    rng = np.random.default_rng(5)
    npages = 9000
    ids = rng.permutation(npages)
    lens = rng.integers(0, 90, n)
    table = np.full((n, 4), -1, np.int32)
    at = 0
    for b in range(n):
        if b and rng.random() < 0.4:
            lens[b], table[b] = lens[b - 1], table[b - 1]
            continue
        h = -(-int(lens[b]) // 32)
        table[b, :h] = ids[at:at + h]
        at += h
    p = Pool(vs, npages, table, lens, layers=1, kv=1)
    assert p.extend([int(c) for c in rng.integers(0, 38, n)]) is None
    p.cache.check()
    p.agrees()
    p.fork([int(x) for x in rng.integers(-1, n, 2000)])
    p.cache.check()
    p.agrees()
    assert p.extend(1) is None
    p.cache.check()
    p.agrees()


def test_a_search_in_beams(vs):
    """Random forks, extensions, evictions and compactions in a row."""
    rng = np.random.default_rng(9)
    p = Pool(vs, 60, rows(6, [3, 8], [3, 8], [3, 20], [5]), [45, 45, 64, 1])
    for step in range(40):
        if rng.random() < 0.3:
            p.fork([int(x) for x in rng.integers(0, 4, 4)])
        if p.model.lens.max() < 180:
            assert p.extend(int(rng.integers(1, 9))) is None
        p.agrees()
        if step % 9 == 8:
            p.cache.compact(p.seqs)
            p.model = p.model.compact()
        p.cache.check()
        p.agrees()


def test_empty_calls(vs):
    p = Pool(vs, 4, np.zeros((0, 3)), [])
    for f in (lambda: p.cache.extend(p.seqs, 1), lambda: p.cache.free(p.seqs), lambda: p.cache.evict(p.seqs, 4),
              lambda: p.cache.compact(p.seqs), lambda: p.extend(0)):
        f()
    p.cache.check()
