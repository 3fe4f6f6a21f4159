"""Calls behind an extend that did not fit: nothing of the cache is lost, nobody else's calls are touched, and
vs_kv_check tells."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu

KV, DIM, HEADS, LAYERS, PAGE = 2, 32, 4, 2, 32


class Cache:
    def __init__(self, vs, npages, table, lens, dtype, seed=0):
        self.vs, self.dtype, self.rng = vs, dtype, np.random.default_rng(seed)
        A = vs.DeviceArray
        some, _ = D.stored(self.rng.standard_normal((min(npages, 61), LAYERS, 2, KV, PAGE * DIM)), dtype)
        self.bits = some[np.arange(npages) % 61]
        self.mem = A.of(self.bits, dtype)
        self.cache = vs.PagedKVCache(npages, PAGE, KV, DIM, layers=LAYERS, dtype=dtype, memory=self.mem)
        table = np.array(table, np.int32)
        refs = np.bincount(table[table >= 0], minlength=npages)
        self.refs = A.of(refs, "i32")
        self.seqs = self.on(table, lens)

    def on(self, table, lens):
        A = self.vs.DeviceArray
        return self.vs.KVSequences(A.of(table, "i32"), A.of(lens, "i32"), self.refs)

    def rows(self, n, heads=KV):
        return D.stored(self.rng.standard_normal((n, heads, DIM)), self.dtype)

    def step(self, seqs):
        """Every layer's attention with a new token, and a row appended; the outputs, the queries and the token."""
        A, n, got = self.vs.DeviceArray, seqs.n, []
        for layer in range(LAYERS):
            (qb, q), (kb, k), (vb, v) = self.rows(n, HEADS), self.rows(n), self.rows(n)
            out = A((n, HEADS, DIM), self.dtype)
            self.cache.attend(seqs, A.of(qb, self.dtype), out, k=A.of(kb, self.dtype), v=A.of(vb, self.dtype), layer=layer)
            o = out.numpy()
            got.append((D.from_bf16(o) if self.dtype == "bf16" else o, q.astype(np.float64), kb, vb))
        return got

    def append(self, seqs, count):
        A, rows = self.vs.DeviceArray, count * seqs.n
        kb, vb = self.rows(rows)[0], self.rows(rows)[0]
        starts = A.of(np.arange(seqs.n + 1) * count, "i32")
        self.cache.append(seqs, A.of(kb, self.dtype), A.of(vb, self.dtype), starts=starts, layer=1)
        return kb, vb

    def same(self):
        assert np.array_equal(self.mem.numpy().view(np.uint16), self.bits.view(np.uint16))

    def old_answers(self, seqs, got):
        """The outputs are the attention over what the cache holds: no new token among it."""
        table, lens = seqs.table.numpy(), seqs.lens.numpy()
        kp, vp = D.places(DIM, self.dtype)
        val = D.from_bf16(self.bits) if self.dtype == "bf16" else self.bits
        for layer, (out, q, _, _) in enumerate(got):
            for b in range(seqs.n):
                rows = [[val[table[b, p // PAGE], layer, kv][:, place[p % 32]] for p in range(lens[b])]
                        for kv, place in ((0, kp), (1, vp))]
                k, v = (np.array(r, np.float64).reshape(-1, KV, DIM) for r in rows)
                args = (q[b], k, v, np.arange(lens[b]), DIM ** -0.5)
                D.assert_rounded(out[b], D.attend(*args)[0], D.attend_tolerance(*args, self.dtype)[0], self.dtype)


def held(c, seqs, layer, b, pos):
    """Keys and values at a position, as stored."""
    A = c.vs.DeviceArray
    k, v = A((1, KV, DIM), c.dtype), A((1, KV, DIM), c.dtype)
    c.cache.read(seqs, b, int(pos), k, v, layer=layer)
    return k.numpy()[0], v.numpy()[0]


# two beams of one parent, whose shared page the refused plan would have copied, and one of its own
PAGES = dict(npages=5, table=[[0, 1, -1], [0, 1, -1], [2, 3, 4]], lens=[40, 40, 70], count=1)
# one past its columns, the others not
COLUMNS = dict(npages=9, table=[[0, 1, -1], [0, 1, -1], [2, 3, 4]], lens=[40, 40, 90], count=7)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [PAGES, COLUMNS])
def test_nothing_is_stored_behind_a_refused_extend(vs, dtype, case):
    c = Cache(vs, case["npages"], case["table"], case["lens"], dtype)
    c.cache.extend(c.seqs, case["count"])
    got = c.step(c.seqs)
    c.append(c.seqs, case["count"])
    assert c.seqs.lens.numpy().tolist() == case["lens"] and c.seqs.table.numpy().tolist() == case["table"]
    c.same()
    c.old_answers(c.seqs, got)
    with pytest.raises((vs.VsError, ValueError)):
        c.cache.check()
    c.cache.check()  # told once


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("npages", [11, 17000])
def test_forks_and_compaction_behind_it(vs, dtype, npages):
    """The beams go on and the cache is compacted before anyone asks: still nothing is lost."""
    top = npages - 1
    c = Cache(vs, npages, [[0, 1, -1], [0, top, -1], [2, 3, 4]], [40, 45, 90], dtype)
    c.cache.extend(c.seqs, 7)  # the third has 96 positions of 96
    spare = c.on(np.full((4, 3), -1, np.int32), np.zeros(4, np.int32))
    c.cache.fork(c.seqs, vs.DeviceArray.of([1, 1, 2, 0], "i32"), spare)
    c.step(spare)
    c.append(spare, 3)
    c.same()
    c.cache.compact(spare)
    c.bits[5] = c.bits[top]  # (the first six pages are in use, and this one moved)
    c.old_answers(spare, c.step(spare))
    c.append(spare, 3)
    c.same()
    with pytest.raises(ValueError, match="table row"):
        c.cache.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_others_go_on(vs, dtype):
    """Another set of sequences on the same cache, extended before the refusal: its new token is stored."""
    c = Cache(vs, 6, [[0, 1, -1], [2, 3, 4]], [40, 70], dtype)
    other = c.on(np.array([[-1, -1]]), np.zeros(1, np.int32))
    c.cache.extend(other, 1)   # the last free page
    c.cache.extend(c.seqs, 26)  # one more wanted, none there
    before = c.mem.numpy().copy()
    got = c.step(other)
    for layer, (_, _, kb, vb) in enumerate(got):
        k, v = held(c, other, layer, 0, 0)
        assert np.array_equal(k, kb[0]) and np.array_equal(v, vb[0])
    after = c.mem.numpy()
    assert np.array_equal(after[:5].view(np.uint16), before[:5].view(np.uint16))
    with pytest.raises(vs.VsError, match="short"):
        c.cache.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("told", [False, True])
def test_an_extend_that_fits_goes_on(vs, dtype, told):
    """Room made and the same sequences extended, with or without a check between: tokens are stored again."""
    c = Cache(vs, 5, [[0, 1, -1], [0, 1, -1], [2, 3, 4]], [40, 40, 70], dtype)
    c.cache.extend(c.seqs, 1)
    c.step(c.seqs)
    c.same()
    if told:
        with pytest.raises(vs.VsError, match="1 pages short"):
            c.cache.check()
    c.cache.free(c.seqs, vs.DeviceArray.of([2], "i32"))
    c.cache.extend(c.seqs, vs.DeviceArray.of([1, 1, 0], "i32"))
    lens = c.seqs.lens.numpy()
    assert lens.tolist() == [41, 41, 0]
    for layer, (_, _, kb, vb) in enumerate(c.step(c.seqs)):
        for b in (0, 1):
            k, v = held(c, c.seqs, layer, b, 40)
            assert np.array_equal(k, kb[b]) and np.array_equal(v, vb[b])
    kb, vb = c.append(c.seqs, 1)
    assert all(np.array_equal(held(c, c.seqs, 1, b, 40)[0], kb[b]) for b in (0, 1))
    if not told:
        with pytest.raises(vs.VsError, match="1 pages short"):
            c.cache.check()
    c.cache.check()


def test_more_sequences_than_one_plan_keeps_in_registers(vs):
    n = 1100
    c = Cache(vs, n, np.arange(n)[:, None], np.full(n, 5), "bf16")
    c.cache.extend(c.seqs, 28)
    c.step(c.seqs)
    c.append(c.seqs, 2)
    c.same()
    with pytest.raises(ValueError, match="table row"):
        c.cache.check()
    c.cache.extend(c.seqs, 27)
    kb, vb = c.append(c.seqs, 2)
    c.cache.check()
    for b in (0, 1023, 1024, n - 1):
        k, v = held(c, c.seqs, 1, b, 31)
        assert np.array_equal(k, kb[2 * b + 1]) and np.array_equal(v, vb[2 * b + 1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_full_page_that_others_end_in_too(vs, dtype):
    """Two sets go on from one full page of a prompt; one is refused, the other's extend does not open that page."""
    c = Cache(vs, 4, [[0, -1]], [32], dtype)
    narrow = c.on(np.array([[0]]), [32])
    c.cache.extend(narrow, 1)  # no column for it
    c.cache.extend(c.seqs, 1)
    before = c.mem.numpy()[0].copy()
    c.step(narrow)
    c.append(narrow, 1)
    for layer, (_, _, kb, vb) in enumerate(c.step(c.seqs)):
        k, v = held(c, c.seqs, layer, 0, 32)
        assert np.array_equal(k, kb[0]) and np.array_equal(v, vb[0])
    assert np.array_equal(c.mem.numpy()[0].view(np.uint16), before.view(np.uint16))
    with pytest.raises(ValueError, match="table row"):
        c.cache.check()
