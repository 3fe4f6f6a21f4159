"""Attention of one new token over the paged cache against its formula in 64
bits: lengths, masks, layouts and types where it can go wrong."""
import numpy as np
import pytest

import _decode as D
from _hip import Stream

pytestmark = pytest.mark.gpu


class View:
    """A strided view of a DeviceArray, as a fused projection's output is one."""

    def __init__(self, base, shape, stride, offset=0):
        self.base, self.shape, self._stride, self.offset, self.dtype = base, shape, stride, offset, base.dtype

    def data_ptr(self):
        return self.base.data_ptr() + int(self.offset * 2) * (1 if self.dtype == "bf16" else 2)

    def stride(self):
        return self._stride


class Case:
    def __init__(self, vs, lens, heads, kv, dim, page=32, dtype="bf16", layers=1, layer=0, width=None, seed=0,
                 spread=1.0):
        rng = np.random.default_rng(seed)
        self.vs, self.lens, self.heads, self.kv, self.dim, self.page = vs, np.array(lens, np.int32), heads, kv, dim, page
        self.dtype, self.layer = dtype, layer
        held = [-(-int(n) // page) for n in lens]
        npages = sum(held) + 3
        ids = rng.permutation(npages)[:sum(held)].astype(np.int32)
        self.table = np.full((len(lens), width or max(held + [1]) + 1), -1, np.int32)
        at = 0
        for b, h in enumerate(held):
            self.table[b, :h] = ids[at:at + h]
            at += h
        # what no position uses holds NaNs
        nan = D.stored(np.full(1, np.nan), dtype)[0][0]
        self.pool = np.full((npages, layers, 2, kv, page * dim), nan, np.uint16 if dtype == "bf16" else np.float32)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            kb, k = D.stored(rng.standard_normal((n, kv, dim)), dtype)
            vb, v = D.stored(rng.standard_normal((n, kv, dim)), dtype)
            D.write_rows(self.pool[:, layer], self.table, b, 0, kb, vb, page, dtype)
            self.k.append(k.astype(np.float64))
            self.v.append(v.astype(np.float64))
        self.qb, q = D.stored(spread * rng.standard_normal((len(lens), heads, dim)), dtype)
        self.q = q.astype(np.float64)
        self.mem = vs.DeviceArray.of(self.pool, dtype)
        self.cache = vs.PagedKVCache(npages, page, kv, dim, layers=layers, dtype=dtype, memory=self.mem)
        self.sequences(np.zeros(npages, np.int32))
        self.rng = rng

    def sequences(self, refs):
        A = self.vs.DeviceArray
        self.seqs = self.vs.KVSequences(A.of(self.table, "i32"), A.of(self.lens, "i32"), A.of(refs, "i32"))

    def run(self, q=None, **kw):
        A = self.vs.DeviceArray
        n = len(self.lens)
        # (poisoned: every value has to be written)
        out = A.of(np.full((n, self.heads, self.dim), 0x7FC1 if self.dtype == "bf16" else 77.0), self.dtype)
        lse = A.of(np.full((n, self.heads), 77.0), "f32")
        self.cache.attend(self.seqs, A.of(self.qb, self.dtype) if q is None else q, out, lse=lse, layer=self.layer, **kw)
        self.cache.check()
        o = out.numpy()
        return (D.from_bf16(o) if self.dtype == "bf16" else o), lse.numpy()

    def compare(self, got, window=0, sinks=0, scale=None, hidden=lambda b, p: np.zeros(len(p), bool)):
        out, lse = got
        scale = self.dim ** -0.5 if scale is None else scale
        for b, n in enumerate(self.lens):
            seen = D.visible(int(n), window, sinks)
            seen = seen[~hidden(b, seen)]
            eo, el = D.attend(self.q[b], self.k[b], self.v[b], seen, scale)
            to, tl = D.attend_tolerance(self.q[b], self.k[b], self.v[b], seen, scale, self.dtype)
            D.assert_rounded(out[b], eo, to, self.dtype, f"sequence {b} of length {n}")
            if len(seen):
                np.testing.assert_allclose(lse[b], el, rtol=0, atol=tl, err_msg=f"sequence {b} of {n}")
            else:
                assert (lse[b] == -np.inf).all()


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 517]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_lengths(vs, dtype, page):
    c = Case(vs, LENGTHS, 8, 2, 64, page, dtype)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", range(16, 257, 16))
def test_head_dims(vs, dtype, dim):
    c = Case(vs, [1, 45, 200], 6, 2, dim, 32, dtype)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (3, 1), (15, 1), (16, 1), (17, 1), (40, 1), (64, 2), (33, 3)])
def test_head_layouts(vs, dtype, heads, kv):
    c = Case(vs, [7, 130], heads, kv, 32, 32, dtype)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (32, 0), (33, 33), (64, 40), (100, 300), (1000, 3),
                                          (2**31 - 1, 2**31 - 1)])
def test_window_and_sinks(vs, dtype, window, sinks):
    c = Case(vs, LENGTHS + [1500], 4, 2, 48, 32, dtype)
    c.compare(c.run(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_missing_pages_are_not_visible(vs, dtype):
    """-1 and ids past the cache: no page, whatever the length says; lengths past the table end there."""
    c = Case(vs, [100, 200, 64, 64], 4, 2, 64, 32, dtype)
    c.table[0, 1] = -1
    c.table[1, [0, 6]] = [c.cache.npages, -7]  # its last positions among them
    c.table[2, :2] = [2**31 - 1, -2**31]       # nothing left
    gone = [set(range(32, 64)), set(range(32)) | set(range(192, 200)), set(range(64)), set()]
    c.sequences(np.zeros(c.cache.npages, np.int32))
    hidden = lambda b, p: np.array([int(x) in gone[b] for x in p], bool)  # noqa: E731
    c.compare(c.run(), hidden=hidden)
    lens = c.lens.copy()
    c.lens = np.array([100, 200, 64, 5000], np.int32)
    c.sequences(np.zeros(c.cache.npages, np.int32))
    out = c.run()
    c.lens = lens
    c.compare(out, hidden=hidden)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_negative_length_is_empty(vs, dtype):
    c = Case(vs, [40, 0], 2, 1, 32, 32, dtype)
    true, c.lens = c.lens, np.array([40, -5], np.int32)
    c.sequences(np.zeros(c.cache.npages, np.int32))
    got = c.run()
    c.lens = true
    c.compare(got)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_length_past_the_table(vs, dtype):
    """A new token without a column is stored nowhere and told; the positions that have one are attended to."""
    c = Case(vs, [64, 70], 4, 2, 32, 32, dtype, width=3)
    true, c.lens = c.lens, np.array([97, 70], np.int32)
    c.table[0, 2] = c.table[0, 0]  # (a page in every column: 96 positions, the first 32 of them twice)
    c.sequences(np.zeros(c.cache.npages, np.int32))
    A = vs.DeviceArray
    n, before = 2, c.mem.numpy().copy()
    kb, _ = D.stored(np.full((n, 2, 32), 3.0), dtype)
    out, lse = A((n, 4, 32), dtype), A((n, 4), "f32")
    c.cache.attend(c.seqs, A.of(c.qb, dtype), out, k=A.of(kb, dtype), v=A.of(kb, dtype), lse=lse)
    with pytest.raises(ValueError, match="outgrew"):
        c.cache.check()
    after = c.mem.numpy()
    changed = {int(p) for p in np.nonzero((before.view(np.uint8) != after.view(np.uint8))
                                          .reshape(len(before), -1).any(1))[0]}
    assert changed == {int(c.table[1, 2])}
    k0, v0 = np.concatenate([c.k[0], c.k[0][:32]]), np.concatenate([c.v[0], c.v[0][:32]])
    args = (c.q[0], k0, v0, np.arange(96), 32 ** -0.5)
    got = D.from_bf16(out.numpy()) if dtype == "bf16" else out.numpy()
    D.assert_rounded(got[0], D.attend(*args)[0], D.attend_tolerance(*args, dtype)[0], dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,heads,n", [(1, 4, 40_000), (1, 16, 9_001), (2, 6, 70_000)])
def test_split_over_the_length(vs, dtype, kv, heads, n):
    """Hundreds of work items of one sequence (more than a wave's lanes), beside a short one."""
    c = Case(vs, [n, 3], heads, kv, 32, 128, dtype, spread=2.0)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("width", [1, 4, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 66])
@pytest.mark.parametrize("dim,n", [(64, 1), (64, 40), (144, 2)])
def test_short_tables_are_not_split(vs, dtype, width, dim, n):
    """Around the table widths where a sequence is one work item, of four waves or eight, with every length."""
    lens = [(7 * i * i + 3) % (32 * width + 1) for i in range(n - 1)] + [32 * width]
    c = Case(vs, lens, 24, 8, dim, 32, dtype, width=width)
    c.compare(c.run())
    c.compare(c.run(window=300, sinks=33), 300, 33)


def test_many_ragged_sequences(vs):
    """More sequences than lanes; empty ones among them."""
    lens = [(i * 37) % 150 if i % 7 else 0 for i in range(333)] + [2000]
    c = Case(vs, lens, 2, 1, 32, 32, "bf16")
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("spread,scale", [(40.0, None), (1.0, 0.0), (1.0, -3.0), (1e-3, 1.0)])
def test_peaked_and_flat(vs, dtype, spread, scale):
    c = Case(vs, [1, 333], 4, 2, 64, 32, dtype, spread=spread)
    c.compare(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0, 1, 2, 8])
def test_strides_and_alignment(vs, dtype, shift):
    """q, k and v as slices of one projection row, at odd offsets; out in rows of its own stride;
    the new token is stored at the last position and nowhere else."""
    H, kv, dim, lens = 6, 3, 48, [1, 32, 33, 100, 64, 0]
    c = Case(vs, lens, H, kv, dim, 32, dtype, layers=3, layer=1)
    n, row = len(lens), (H + 2 * kv) * dim + shift
    bits, x = D.stored(c.rng.standard_normal(n * row + shift), dtype)
    buf = vs.DeviceArray.of(bits, dtype)
    x = np.concatenate([x[shift:].astype(np.float64), np.zeros(shift)])
    cut = lambda a, o, h: np.stack([a[b * row + o * dim:][:h * dim].reshape(h, dim) for b in range(n)])  # noqa: E731
    view = lambda o, h: View(buf, (n, h, dim), (row, dim, 1), shift + o * dim)  # noqa: E731
    c.q = cut(x, 0, H)
    raw = np.concatenate([bits[shift:], np.zeros(shift, bits.dtype)])
    c.qb, kb, vb = cut(raw, 0, H), cut(raw, H, kv), cut(raw, H + kv, kv)
    orow = H * dim + 5
    obuf = vs.DeviceArray.of(np.full((n, orow), 3), dtype)
    c.cache.attend(c.seqs, view(0, H), View(obuf, (n, H, dim), (orow, dim, 1)), k=view(H, kv), v=view(H + kv, kv), layer=1)
    for b, ln in enumerate(lens):
        if ln:
            c.k[b][-1], c.v[b][-1] = cut(x, H, kv)[b], cut(x, H + kv, kv)[b]
            D.write_rows(c.pool[:, 1], c.table, b, ln - 1, kb[b:b + 1], vb[b:b + 1], 32, dtype)
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))
    o = obuf.numpy()
    assert (o[:, H * dim:] == 3).all()
    o = (D.from_bf16(o) if dtype == "bf16" else o)[:, :H * dim].reshape(n, H, dim)
    lse = c.run()[1]
    c.compare((o, lse))
    assert np.array_equal(c.run()[0], o)  # and from the stored token, to the bit


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 128), (40, 1, 80), (4, 2, 256)])
def test_new_token_at_every_place(vs, dtype, heads, kv, dim):
    """The fused store at all 32 places of a block, windows and groups of more than 16 heads."""
    lens = list(range(1, 33)) + [64, 65, 97]
    c = Case(vs, lens, heads, kv, dim, 32, dtype)
    kb, k = D.stored(c.rng.standard_normal((len(lens), kv, dim)), dtype)
    vb, v = D.stored(c.rng.standard_normal((len(lens), kv, dim)), dtype)
    A = vs.DeviceArray
    got = c.run(k=A.of(kb, dtype), v=A.of(vb, dtype), window=40, sinks=2)
    for b, n in enumerate(lens):
        c.k[b][-1], c.v[b][-1] = k[b], v[b]
        D.write_rows(c.pool[:, 0], c.table, b, n - 1, kb[b:b + 1], vb[b:b + 1], 32, dtype)
    c.compare(got, 40, 2)
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinities_and_nans_show(vs, dtype):
    """A NaN that is visible makes its heads NaN and no others; one value of +-inf goes where it belongs."""
    c = Case(vs, [50, 50, 50], 4, 2, 32, 32, dtype)
    nan, inf = D.stored(np.array([np.nan, np.inf]), dtype)[0]
    kp, vp = D.places(32, dtype)
    c.pool[c.table[0, 0], 0, 0, 1, kp[5, 3]] = nan           # a key of sequence 0, kv head 1
    c.pool[c.table[1, 1], 0, 1, 0, 0 + vp[40 % 32, 7]] = inf  # a value of sequence 1, kv head 0, dimension 7
    c.mem.upload(c.pool)
    out, lse = c.run()
    assert np.isnan(out[0, 2:]).all() and np.isnan(lse[0, 2:]).all() and np.isfinite(out[0, :2]).all()
    assert (out[1, :2, 7] == np.inf).all()
    rest = np.ones((4, 32), bool)
    rest[:2, 7] = False
    assert np.isfinite(out[1][rest]).all() and np.isfinite(out[2]).all()
    hidden, _ = c.run(window=9)
    assert np.isfinite(hidden[0]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinite_value_alone(vs, dtype):
    """One position, weight 1: its values come back as they are, infinities too."""
    c = Case(vs, [1], 2, 1, 32, 32, dtype)
    inf = D.stored(np.array([np.inf, -np.inf]), dtype)[0]
    vp = D.places(32, dtype)[1]
    c.pool[c.table[0, 0], 0, 1, 0, vp[0, :2]] = inf
    c.mem.upload(c.pool)
    out, _ = c.run()
    assert (out[0, :, 0] == np.inf).all() and (out[0, :, 1] == -np.inf).all()
    assert np.array_equal(out[0, :, 2:], np.tile(c.v[0][0, :, 2:], (2, 1)))


def test_refusals(vs):
    c = Case(vs, [5, 6], 4, 2, 32, 32, "bf16")
    A = vs.DeviceArray
    q, out, k = A((2, 4, 32), "bf16"), A((2, 4, 32), "bf16"), A((2, 2, 32), "bf16")
    for bad in (dict(layer=1), dict(layer=-1), dict(window=-1), dict(sinks=-1), dict(k=k), dict(k=k, v=A((2, 2, 48), "bf16")),
                dict(scale=float("nan")), dict(lse=A((2, 4), "bf16")), dict(lse=A((4, 2), "f32"))):
        with pytest.raises(ValueError):
            c.cache.attend(c.seqs, q, out, **bad)
    with pytest.raises(ValueError, match="multiple"):
        c.cache.attend(c.seqs, A((2, 3, 32), "bf16"), A((2, 3, 32), "bf16"))
    with pytest.raises(ValueError):
        c.cache.attend(c.seqs, A((2, 4, 32), "f32"), out)
    with pytest.raises(ValueError):
        c.cache.attend(c.seqs, q, A((3, 4, 32), "bf16"))
    with pytest.raises(ValueError, match="pages"):
        c.cache.attend(vs.KVSequences(c.seqs.table, c.seqs.lens, A((c.cache.npages + 1,), "i32")), q, out)
    with pytest.raises(ValueError):
        c.cache.append(c.seqs, A((3, 2, 32), "bf16"), A((3, 2, 32), "bf16"))  # no starts, three rows
    with pytest.raises(ValueError, match="sequence 2"):
        c.cache.read(c.seqs, 2, 0, k, k)
    with pytest.raises(ValueError, match="window"):
        c.cache.evict(c.seqs, 0)
    with pytest.raises(ValueError, match="another table"):
        c.cache.fork(c.seqs, A((2,), "i32"), c.seqs)
    with pytest.raises(ValueError, match="aligned"):
        c.cache.attend(c.seqs, View(q, (2, 4, 32), (0, 0, 1), 0.5), out)
    with pytest.raises(NotImplementedError, match="head_dim"):
        vs.PagedKVCache(4, 32, 1, 40)
    with pytest.raises(ValueError, match="values"):
        vs.PagedKVCache(400, 32, 1, 32, memory=q)
    c.compare(c.run())  # still sound


def test_same_bits_every_time_and_alone(vs):
    """No atomics, no order: runs agree to the bit."""
    c = Case(vs, [3000, 17, 900, 5000], 8, 2, 64, 32, "bf16")
    first = c.run()
    for _ in range(3):
        again = c.run()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_cache_past_four_gib(vs):
    """Pages whose offsets pass 32 bits."""
    page, kv, dim = 1024, 4, 128
    npages = (5 << 30) // (2 * kv * page * dim * 2)
    cache = vs.PagedKVCache(npages, page, kv, dim)
    A = vs.DeviceArray
    rng = np.random.default_rng(3)
    n = 1500
    table = np.array([[npages - 1, npages - 2]], np.int32)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of([n], "i32"), A.of(np.zeros(npages, np.int32), "i32"))
    kb, k = D.stored(rng.standard_normal((n, kv, dim)), "bf16")
    vb, v = D.stored(rng.standard_normal((n, kv, dim)), "bf16")
    cache.append(seqs, A.of(kb, "bf16"), A.of(vb, "bf16"), starts=A.of([0, n], "i32"))
    qb, q = D.stored(rng.standard_normal((1, 8, dim)), "bf16")
    out = A((1, 8, dim), "bf16")
    cache.attend(seqs, A.of(qb, "bf16"), out)
    cache.check()
    args = (q[0].astype(np.float64), k.astype(np.float64), v.astype(np.float64), np.arange(n), dim ** -0.5)
    D.assert_rounded(D.from_bf16(out.numpy())[0], D.attend(*args)[0], D.attend_tolerance(*args, "bf16")[0], "bf16")
    ko, vo = A((n, kv, dim), "bf16"), A((n, kv, dim), "bf16")
    cache.read(seqs, 0, 0, ko, vo)
    assert np.array_equal(ko.numpy(), kb) and np.array_equal(vo.numpy(), vb)
    cache.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_as_many_positions_as_a_length_counts(vs, dtype):
    """Positions near 2^31, in a table that names one page over and over: weights and values of one, whose sums
    are whole numbers and exact but for the join of some 600 items in 32 bits, log sum exp is log n."""
    page, dim = 1024, 16
    cache = vs.PagedKVCache(1, page, 1, dim, dtype=dtype)
    A = vs.DeviceArray
    one = D.stored(np.ones((page, 1, dim)), dtype)[0]
    first = vs.KVSequences(A.of([[0]], "i32"), A.of([page], "i32"), A.of([1], "i32"))
    cache.append(first, A.of(one, dtype), A.of(one, dtype), starts=A.of([0, page], "i32"))
    q = A.of(D.stored(np.zeros((1, 2, dim)), dtype)[0], dtype)
    for n in (2 ** 29 + 33, 2 ** 31 - 1024 - 33):
        seqs = vs.KVSequences(A.of(np.zeros((1, -(-n // page)), np.int32), "i32"), A.of([n], "i32"), A.of([1], "i32"))
        out, lse = A((1, 2, dim), dtype), A((1, 2), "f32")
        cache.attend(seqs, q, out, lse=lse)
        cache.check()
        o = D.from_bf16(out.numpy()) if dtype == "bf16" else out.numpy()
        tol = 2 * 600 * 2.0 ** -23
        D.assert_rounded(o, np.ones(o.shape), tol, dtype)
        assert np.abs(lse.numpy() - np.log(n)).max() <= tol + 2.0 ** -21 * (np.log(n) + 20)
    cache.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_and_read(vs, dtype):
    """Rows of several sequences to their last positions, and back; positions without a page are dropped and read 0."""
    c = Case(vs, [70, 0, 33, 128, 5], 2, 2, 48, 32, dtype, layers=2, layer=1)
    counts = [40, 0, 1, 97, 5]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = int(starts[-1])
    c.table[3, 2] = -1
    c.sequences(np.zeros(c.cache.npages, np.int32))
    kb, _ = D.stored(c.rng.standard_normal((rows, 2, 48)), dtype)
    vb, _ = D.stored(c.rng.standard_normal((rows, 2, 48)), dtype)
    A = vs.DeviceArray
    c.cache.append(c.seqs, A.of(kb, dtype), A.of(vb, dtype), starts=A.of(starts, "i32"), layer=1)
    c.cache.check()
    for b, (n, ln) in enumerate(zip(counts, c.lens)):
        for j in range(n):
            if c.table[b, (ln - n + j) // 32] >= 0:
                at = starts[b] + j
                D.write_rows(c.pool[:, 1], c.table, b, ln - n + j, kb[at:at + 1], vb[at:at + 1], 32, dtype)
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))
    ko, vo = A((128, 2, 48), dtype), A((128, 2, 48), dtype)
    c.cache.read(c.seqs, 3, 0, ko, vo, layer=1)
    want = kb[starts[3]:starts[4]].copy()
    got = ko.numpy()[128 - 97:]
    missing = np.array([p // 32 == 2 for p in range(128 - 97, 128)])
    assert np.array_equal(got[~missing], want[~missing]) and not got[missing].any()
    one = A((5, 2, 48), dtype)
    c.cache.append(c.seqs, one, one, layer=1)  # without starts: one row each
    c.cache.check()


@pytest.mark.parametrize("dtype,dim,shift", [("bf16", 128, 0), ("bf16", 80, 3), ("f32", 256, 0), ("f32", 16, 1)])
def test_append_at_every_offset(vs, dtype, dim, shift):
    """Rows that start and end anywhere in a block, sequences of every small count, from a strided buffer;
    positions before 0, rows outside the buffer and everything else in the pool stay as they were."""
    counts = [n for n in range(0, 40)] + [64, 65, 95, 97, 130]
    lens = [n + (7 * n) % 45 for n in counts]
    lens[5] = 3  # fewer positions than rows: the first two rows have none
    c = Case(vs, lens, 2, 2, dim, 64, dtype, layers=2, layer=1)
    starts = 4 + np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = int(starts[-1]) - 2  # (the last two rows are not there)
    A = vs.DeviceArray
    wide = 5 * dim + 3
    flat, _ = D.stored(c.rng.standard_normal(shift + rows * wide), dtype)
    buf = A.of(flat, dtype)
    at = flat[shift:].reshape(rows, wide)
    k = View(buf, (rows, 2, dim), (wide, dim, 1), shift)
    v = View(buf, (rows, 2, dim), (wide, dim, 1), shift + 3 * dim)
    c.cache.append(c.seqs, k, v, starts=A.of(starts, "i32"), layer=1)
    c.cache.check()
    for b, (n, ln) in enumerate(zip(counts, lens)):
        for j in range(n):
            p, r = ln - n + j, int(starts[b]) + j
            if p >= 0 and r < rows:
                D.write_rows(c.pool[:, 1], c.table, b, p, at[r, :2 * dim].reshape(1, 2, dim),
                             at[r, 3 * dim:5 * dim].reshape(1, 2, dim), 64, dtype)
    assert np.array_equal(c.mem.numpy().view(np.uint16), c.pool.view(np.uint16))


def test_streams_have_scratch_of_their_own(vs):
    """One handle, three streams at a time, split work on each."""
    c = Case(vs, [4000, 9], 4, 1, 64, 32, "bf16")
    want = c.run()
    A = vs.DeviceArray
    q = A.of(c.qb, "bf16")
    outs = [(A.of(np.zeros((2, 4, 64)), "bf16"), A.of(np.zeros((2, 4)), "f32"), s)
            for s in [Stream() for _ in range(3)] for _ in range(8)]
    for out, lse, s in outs[::8] + outs:
        c.cache.attend(c.seqs, q, out, lse=lse, stream=s.ptr)
    for _, _, s in outs:
        s.sync()
    for out, lse, _ in outs:
        assert np.array_equal(D.from_bf16(out.numpy()), want[0]) and np.array_equal(lse.numpy(), want[1])


def test_recorded_into_a_graph(vs):
    """A decoding step recorded once and replayed with other contents and eager calls between; a call that would
    have to allocate while it is recorded is refused."""
    c = Case(vs, [90, 31, 64], 4, 2, 64, 32, "bf16", width=300)  # room for sequences that have to be split
    refs = np.bincount(c.table[c.table >= 0], minlength=c.cache.npages).astype(np.int32)
    c.sequences(refs)
    A = vs.DeviceArray
    q, out, st = A.of(c.qb, "bf16"), A.of(np.zeros((3, 4, 64)), "bf16"), Stream()
    other = c.cache.new_sequences(3, 300)
    parents = A.of([2, 1, 0], "i32")

    def step():
        c.cache.attend(c.seqs, q, out, stream=st.ptr)
        c.cache.fork(c.seqs, parents, other, stream=st.ptr)
        c.cache.extend(other, 1, stream=st.ptr)

    st.begin()
    try:
        with pytest.raises(NotImplementedError, match="scratch"):
            c.cache.attend(c.seqs, q, out, stream=st.ptr)
        c.cache.fork(c.seqs, parents, other, stream=st.ptr)
    finally:
        st.end()
    step()  # scratch of this size exists now
    st.sync()
    st.begin()
    step()
    graph = st.end()
    for i in range(5):
        c.qb, x = D.stored(c.rng.standard_normal((3, 4, 64)), "bf16")
        c.q = x.astype(np.float64)
        q.upload(c.qb)
        parents.upload(c.rng.permutation(3))
        st.replay(graph)
        got, table, lens = D.from_bf16(out.numpy()), other.table.numpy(), other.lens.numpy()
        c.compare((got, c.run()[1]))
        m = D.Pages(c.table, c.lens, refs, 32).fork(parents.numpy())
        assert m.extend(1) is None
        assert np.array_equal(table, m.table) and np.array_equal(lens, m.lens)
        assert np.array_equal(other.refs.numpy(), m.refs)
    c.cache.check()


def test_failed_allocations(vs):
    """Scratch that cannot be had: the call fails as out of memory, and the next one works; so does a cache."""
    c = Case(vs, [5000, 70], 4, 1, 64, 32, "bf16")
    index = vs.GpuIndexFlat.ip(8)
    for f in (c.run, lambda: c.cache.extend(c.seqs, 1), lambda: vs.PagedKVCache(4, 32, 1, 32)):
        index.set_option("fail_alloc", 1)
        with pytest.raises(vs.VsError, match="memory"):
            f()
    index.set_option("fail_alloc", 0)
    c.compare(c.run())
    vs.PagedKVCache(4, 32, 1, 32).close()
    index.close()
