"""Attention of many new tokens over the paged cache against its formula in 64
bits: lengths, rows, masks, layouts and types where it can go wrong."""
import numpy as np
import pytest

import _decode as D
import _prompt as P
from _hip import Stream
from test_gpu_attend import Case, View

pytestmark = pytest.mark.gpu


class Rows(Case):
    """counts[b] rows for the last positions of sequence b; `lead` rows before them and `tail` behind are no one's."""

    def __init__(self, vs, lens, counts, heads, kv, dim, page=32, dtype="bf16", lead=0, tail=0, spread=1.0, **kw):
        super().__init__(vs, lens, heads, kv, dim, page, dtype, spread=spread, **kw)
        self.counts = np.array(counts)
        self.starts = lead + np.concatenate([[0], self.counts.cumsum()])
        self.nrows = int(self.starts[-1]) + tail
        self.qb, q = D.stored(spread * self.rng.standard_normal((self.nrows, heads, dim)), dtype)
        self.q = q.astype(np.float64)

    def poisoned(self):
        A = self.vs.DeviceArray
        return (A.of(np.full((self.nrows, self.heads, self.dim), 0x7FC1 if self.dtype == "bf16" else 77.0), self.dtype),
                A.of(np.full((self.nrows, self.heads), 77.0), "f32"))

    def values(self, out, lse):
        o = out.numpy()
        return (D.from_bf16(o) if self.dtype == "bf16" else o), lse.numpy()

    def run(self, q=None, **kw):
        A = self.vs.DeviceArray
        out, lse = self.poisoned()
        self.cache.attend_rows(self.seqs, A.of(self.qb, self.dtype) if q is None else q, out, lse=lse, layer=self.layer,
                               starts=A.of(self.starts, "i32"), **kw)
        self.cache.check()
        return self.values(out, lse)

    def compare(self, got, window=0, sinks=0, scale=None, causal=True, missing=lambda b: ()):
        out, lse = got
        scale = self.dim ** -0.5 if scale is None else scale
        kept = np.ones(self.nrows, bool)
        for b, (n, c) in enumerate(zip(self.lens, self.counts)):
            n = max(int(n), 0)
            at = slice(self.starts[b], self.starts[b] + c)
            kept[at] = False
            if c == 0:
                continue
            last = np.arange(n - c, n) if causal else np.full(c, n - 1)
            seen = P.seen_mask(last, len(self.k[b]), window, sinks)
            seen[:, list(missing(b))] = False
            eo, el, to, tl = P.attend_rows(self.q[at], self.k[b], self.v[b], seen, scale, self.dtype)
            D.assert_rounded(out[at], eo, to, self.dtype, f"sequence {b} of length {n}, {c} rows")
            some = np.isfinite(el)
            assert (np.abs(lse[at] - el)[some] <= tl[some]).all(), (b, n, c)
            assert (lse[at][~some] == -np.inf).all()
        # rows of no sequence are left as they were
        assert (np.isnan(out[kept]) if self.dtype == "bf16" else out[kept] == 77.0).all() and (lse[kept] == 77.0).all()


LENS = [0, 1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 300, 517, 40, 9, 7]
ROWS = [0, 1, 1, 31, 7, 33, 64, 2, 1, 128, 100, 0, 200, 3, 9, 5]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_and_rows(vs, dtype, page, causal):
    c = Rows(vs, LENS, ROWS, 4, 2, 64, page, dtype, lead=3, tail=70)
    c.compare(c.run(causal=causal), causal=causal)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", range(16, 257, 16))
def test_head_dims(vs, dtype, dim):
    c = Rows(vs, [1, 45, 200, 170], [1, 45, 50, 3], 6, 2, dim, 32, dtype)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (3, 1), (15, 1), (16, 1), (17, 1), (40, 1), (130, 1), (64, 2), (33, 3)])
def test_head_layouts(vs, dtype, heads, kv):
    c = Rows(vs, [7, 130, 60], [7, 40, 1], heads, kv, 32, 32, dtype, tail=1)
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (32, 0), (33, 33), (64, 40), (100, 300), (1000, 3),
                                          (2**31 - 1, 2**31 - 1)])
def test_window_and_sinks(vs, dtype, window, sinks):
    c = Rows(vs, LENS + [1500], ROWS + [900], 4, 2, 48, 32, dtype)
    c.compare(c.run(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(vs, dtype, scale):
    c = Rows(vs, [70, 200], [70, 20], 4, 2, 64, 32, dtype)
    c.compare(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_before_the_first_position_see_nothing(vs, dtype):
    """More rows than positions, and lengths below 0."""
    c = Rows(vs, [5, 0, 0, 40], [9, 3, 140, 41], 4, 2, 32, 32, dtype)
    c.lens = np.array([5, 0, -7, 40], np.int32)
    c.sequences(np.zeros(c.cache.npages, np.int32))
    c.compare(c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_without_starts_one_row_each(vs, dtype):
    lens = [1, 17, 64, 300, 0]
    c = Rows(vs, lens, [1] * 5, 8, 2, 64, 32, dtype)
    out, lse = c.poisoned()
    c.cache.attend_rows(c.seqs, vs.DeviceArray.of(c.qb, dtype), out, lse=lse)
    c.compare(c.values(out, lse))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
def test_missing_pages_are_not_visible(vs, dtype, causal):
    """-1 and ids past the cache: no page, whatever the length says; lengths past the table end there."""
    c = Rows(vs, [100, 200, 64, 64], [60, 200, 30, 3], 4, 2, 64, 32, dtype)
    c.table[0, 1] = -1
    c.table[1, [0, 6]] = [c.cache.npages, -7]  # the first rows see nothing, the last positions are missing
    c.table[2, :2] = [2**31 - 1, -2**31]       # nothing left
    gone = [range(32, 64), list(range(32)) + list(range(192, 200)), range(64), []]
    c.sequences(np.zeros(c.cache.npages, np.int32))
    c.compare(c.run(causal=causal), causal=causal, missing=lambda b: gone[b])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_may_be_anything(vs, dtype, window, bad):
    """A value that is not finite among the chunk's own: rows before it (and past its window) are as without it,
    rows that see it are not finite there."""
    n, rows, at, dim = 150, 140, 77, 64
    c = Rows(vs, [n, 90], [rows, 90], 4, 2, dim, 32, dtype, spread=0.5)
    free = c.run(window=window)
    page, t = c.table[0, at // 32], at % 32
    _, vp = D.places(dim, dtype)
    c.pool[page, 0, 1, 1, vp[t, 5]] = D.stored(np.full(1, bad), dtype)[0][0]  # dimension 5 of the second key-value head
    c.mem.upload(c.pool)
    out, lse = c.run(window=window)
    last = np.arange(n - rows, n)
    sees = np.concatenate([P.seen_mask(last, n, window, 0)[:, at], np.zeros(90, bool)])
    assert sees.any() and not sees[:rows].all()
    same = np.ones((c.nrows, 4, dim), bool)
    same[sees, 2:, 5] = False
    assert np.array_equal(lse, free[1])
    assert not np.isfinite(out[~same]).any()
    if not np.isnan(bad):
        # (a weight may be too small for 32 bits, and 0 times an infinity is a NaN)
        assert (np.isnan(out[~same]) | (out[~same] == bad)).all() and (out[~same] == bad).mean() > 0.9
    # blocks without a hidden position go through other instructions, whose sums are in another order
    c.v[0][at, 1, 5] = 0
    clean = np.where(same, out, 0)
    want = np.where(same, free[0], 0)
    np.testing.assert_allclose(clean, want, rtol=0, atol=np.abs(want).max() * 2.0 ** (-6 if dtype == "bf16" else -18))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_keys_that_are_not_finite_where_no_one_sees_them(vs, dtype):
    n, rows, at, dim = 150, 140, 100, 64
    c = Rows(vs, [n], [rows], 4, 2, dim, 32, dtype)
    free = c.run()
    kp, _ = D.places(dim, dtype)
    c.pool[c.table[0, at // 32], 0, 0, 0, kp[at % 32, 3]] = D.stored(np.full(1, np.nan), dtype)[0][0]
    c.mem.upload(c.pool)
    out, lse = c.run()
    before = np.arange(n - rows, n) < at
    for got, want in ((out, free[0]), (lse, free[1])):
        assert np.array_equal(got[before], want[before]) and np.array_equal(got[:, 2:], want[:, 2:])
        assert np.isnan(got[~before][:, :2]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strided_rows(vs, dtype, offset):
    """Queries as a part of a projection's output, answers into a part of another buffer; any alignment."""
    A = vs.DeviceArray
    c = Rows(vs, [100, 40], [90, 33], 4, 2, 32, 32, dtype)
    wide, es = 4 * 32 + 51, 2 if dtype == "bf16" else 4
    host = np.zeros((c.nrows + 1, wide), c.qb.dtype)
    host[:c.nrows, offset:offset + 128] = c.qb.reshape(c.nrows, 128)
    base, ob = A.of(host, dtype), A.of(np.full((c.nrows + 1, wide), 9), dtype)
    view = lambda x: View(x, (c.nrows, 4, 32), (wide, 32, 1), offset)  # noqa: E731
    c.cache.attend_rows(c.seqs, view(base), view(ob), starts=A.of(c.starts, "i32"))
    c.cache.check()
    got = ob.numpy()
    rest = np.delete(got[:c.nrows], np.s_[offset:offset + 128], 1)
    assert (rest == 9).all() and (got[c.nrows] == 9).all(), es
    got = got[:c.nrows, offset:offset + 128].reshape(c.nrows, 4, 32)
    _, lse = c.run()
    c.compare(((D.from_bf16(got) if dtype == "bf16" else got), lse))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,counts", [([5000], [3]), ([9000, 100, 4000], [1, 90, 40]), ([3000] * 3, [200, 1, 64]),
                                         ([20000], [20])])
@pytest.mark.parametrize("width", [None, 4000])
def test_few_rows_over_long_sequences(vs, dtype, lens, counts, width):
    """The length is divided among workgroups and joined; the table may be far wider than what is used."""
    c = Rows(vs, lens, counts, 8, 2, 32, 64, dtype, width=width, spread=2.0)
    c.compare(c.run())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [383, 384, 385, 700])
def test_many_sequences(vs, n, causal):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 90, n)
    c = Rows(vs, lens, np.minimum(rng.integers(0, 4, n), lens), 2, 1, 16, 32, "bf16", tail=5)
    c.compare(c.run(causal=causal), causal=causal)


def test_many_tiles(vs):
    """Enough rows that the length is not divided."""
    c = Rows(vs, [700, 300, 1200], [650, 300, 1000], 16, 16, 32, 64, "bf16", tail=3)
    c.compare(c.run())
    c.compare(c.run(window=100, sinks=5), 100, 5)


def test_bounds_of_starts_are_kept(vs):
    """Rows past nrows are left out, and what is there keeps its positions."""
    A = vs.DeviceArray
    c = Rows(vs, [60, 80], [40, 50], 4, 2, 32, 32, "bf16")
    full = c.run()
    cut = 65
    out = A.of(np.full((cut, 4, 32), 0x7FC1), "bf16")
    c.cache.attend_rows(c.seqs, A.of(c.qb[:cut], "bf16"), out, starts=A.of(c.starts, "i32"))
    assert np.array_equal(D.from_bf16(out.numpy()), full[0][:cut])


def test_cache_past_4_gib(vs):
    """Pages whose offsets pass 32 bits."""
    A, dim, kv, page = vs.DeviceArray, 128, 8, 64
    npages = 4200  # of 1 MiB each
    cache = vs.PagedKVCache(npages, page, kv, dim, layers=2, dtype="f32")
    assert npages * cache.page_bytes > 2**32
    rng = np.random.default_rng(0)
    n, c = 150, 100
    table = np.array([[npages - 1, 3, npages - 2]], np.int32)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of([n], "i32"), A.of(np.zeros(npages), "i32"))
    k, v, q = (rng.standard_normal((r, h, dim)).astype(np.float32) for r, h in ((n, kv), (n, kv), (c, kv)))
    cache.append(seqs, A.of(k, "f32"), A.of(v, "f32"), starts=A.of([0, n], "i32"), layer=1)
    out = A((c, kv, dim), "f32")
    cache.attend_rows(seqs, A.of(q, "f32"), out, starts=A.of([0, c], "i32"), layer=1)
    cache.check()
    args = [x.astype(np.float64) for x in (q, k, v)]
    eo, _, to, _ = P.attend_rows(*args, P.seen_mask(np.arange(n - c, n), n, 0, 0), dim ** -0.5, "f32")
    D.assert_rounded(out.numpy(), eo, to, "f32")
    cache.close()


def test_streams_and_graphs(vs):
    """Calls of several sizes on streams of their own, and recorded calls replayed with other work between."""
    A = vs.DeviceArray
    c = Rows(vs, [4000, 300, 900], [5, 100, 70], 8, 2, 64, 32, "bf16")
    want, wl = c.run()
    q, starts = A.of(c.qb, "bf16"), A.of(c.starts, "i32")
    streams = [Stream() for _ in range(3)]
    outs = [[c.poisoned() for _ in range(4)] for _ in streams]
    for st, mine in zip(streams, outs):  # (scratch exists, so that nothing waits below)
        c.cache.attend_rows(c.seqs, q, mine[0][0], lse=mine[0][1], starts=starts, stream=st.ptr)
    for j in range(4):
        for st, mine in zip(streams, outs):
            c.cache.attend_rows(c.seqs, q, mine[j][0], lse=mine[j][1], starts=starts, stream=st.ptr)
    for st, mine in zip(streams, outs):
        st.sync()
        for out, lse in mine:
            got = c.values(out, lse)
            assert np.array_equal(got[0], want) and np.array_equal(got[1], wl)
    st, (out, lse) = streams[0], c.poisoned()
    st.begin()
    c.cache.attend_rows(c.seqs, q, out, lse=lse, starts=starts, stream=st.ptr)
    graph = st.end()
    for i in range(4):
        out.upload(c.poisoned()[0].numpy())
        other = c.run()  # (the program's own work between the replays)
        st.replay(graph)
        assert np.array_equal(c.values(out, lse)[0], want) and np.array_equal(other[0], want)


def test_recording_before_scratch_exists_is_refused(vs):
    A = vs.DeviceArray
    c = Rows(vs, [4000], [5], 8, 2, 64, 32, "bf16")
    q, starts, (out, _), st = A.of(c.qb, "bf16"), A.of(c.starts, "i32"), c.poisoned(), Stream()
    st.begin()
    with pytest.raises(NotImplementedError, match="scratch"):
        c.cache.attend_rows(c.seqs, q, out, starts=starts, stream=st.ptr)
    st.end()
    c.compare(c.run())


def test_refusals(vs):
    A = vs.DeviceArray
    c = Rows(vs, [64], [10], 4, 2, 32, 32, "bf16")
    q, (out, lse), starts = A.of(c.qb, "bf16"), c.poisoned(), A.of(c.starts, "i32")
    call = lambda q=q, out=out, **kw: c.cache.attend_rows(c.seqs, q, out, **{"starts": starts, **kw})  # noqa: E731
    bad = [
        ("window", dict(window=-1)), ("window", dict(sinks=-1)), ("window", dict(window=3, causal=False)),
        ("layer", dict(layer=1)), ("scale", dict(scale=float("nan"))), ("scale", dict(scale=3e38)),
        ("starts", dict(starts=A.of([0], "i32"))), ("starts", dict(starts=A.of([0.0, 1.0], "f32"))),
        ("out", dict(out=A((10, 4, 16), "bf16"))), ("q", dict(q=A((10, 4, 32), "f32"))),
        ("lse", dict(lse=A((10, 3), "f32"))), ("one row per sequence", dict(starts=None)),
        ("multiple", dict(q=A((10, 3, 32), "bf16"), out=A((10, 3, 32), "bf16"))),
    ]
    for word, kw in bad:
        with pytest.raises(ValueError, match=word):
            call(**kw)
    # nothing to do
    c.cache.attend_rows(c.seqs, A((0, 4, 32), "bf16"), A((0, 4, 32), "bf16"), starts=A.of([0, 0], "i32"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [700, 2000])
def test_prompts_in_pieces(vs, dtype, rows):
    """Causal tiles that grow from the first to the last, divided along the length: no piece is left out, whatever
    their numbers go by."""
    c = Rows(vs, [2000, 33], [rows, 33], 2, 1, 32, 64, dtype, tail=1)
    c.compare(c.run())
    c.compare(c.run(window=900, sinks=40), 900, 40)
    c.compare(c.run(causal=False), causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_position_is_answered_by_its_value(vs, dtype):
    """A single weight divided by itself: the value, whatever its score (a reciprocal's rounding, 2^-23, is below half
    a step of bf16)."""
    c = Rows(vs, [70, 200], [70, 150], 4, 2, 48, 32, dtype, spread=3.0)
    out, _ = c.run(window=1)
    for b, (n, r) in enumerate(zip(c.lens, c.counts)):
        want = np.repeat(c.v[b][n - r:], 2, 1)
        got = out[c.starts[b]:c.starts[b + 1]]
        if dtype == "bf16":
            assert np.array_equal(got, want)
        else:
            np.testing.assert_allclose(got, want, rtol=2.0 ** -22, atol=0)


def test_in_place_and_overlaps(vs):
    """Answers may take the queries' place; other overlaps are refused."""
    A = vs.DeviceArray
    for lens, counts in (([300, 70], [200, 70]), ([6000], [9])):  # whole tiles, and tiles in pieces
        c = Rows(vs, lens, counts, 4, 2, 32, 32, "bf16")
        q, starts, want = A.of(c.qb, "bf16"), A.of(c.starts, "i32"), c.run()[0]
        c.cache.attend_rows(c.seqs, q, q, starts=starts)
        assert np.array_equal(D.from_bf16(q.numpy()), want)
    with pytest.raises(ValueError, match="overlaps"):
        c.cache.attend_rows(c.seqs, q, View(q, (9, 4, 32), (128, 32, 1), 8), starts=starts)
    with pytest.raises(ValueError, match="overlaps"):
        c.cache.attend_rows(c.seqs, q, q, starts=starts, lse=LseOver(q, 9, 4))


class LseOver:
    """fp32 over another array's memory."""

    def __init__(self, base, rows, heads):
        self.base, self.shape, self.dtype = base, (rows, heads), "f32"

    def data_ptr(self):
        return self.base.data_ptr()

    def stride(self):
        return (self.shape[1], 1)
