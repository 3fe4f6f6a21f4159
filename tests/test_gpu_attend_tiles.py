"""Attention of many rows in calls that fill the card: tiles of 256 and of 128 rows whose lengths are not divided, against
the formula in 64 bits.  Which kernel a call takes goes by its sizes; the rule stands here again, so that no case drifts
off the kernel it is for."""
import re

import numpy as np
import pytest

import _decode as D
import _prompt as P
from _hip import Stream
from test_gpu_attend_rows import Rows

pytestmark = pytest.mark.gpu


def kernel(vs, nrows, heads, kv, nseq, width, page, dim, dtype):
    """(rows of a tile, whether lengths are divided among workgroups)"""
    cus, group = int(re.search(r"(\d+) CUs", vs.device_name(0)).group(1)), heads // kv
    tiles = lambda tile: nrows * group // tile + nseq  # noqa: E731
    few = nrows * group <= nseq * 64
    prompts = tiles(64) * kv <= 4 * cus and width * page * nseq <= 4 * nrows
    tile = 64
    if dtype == "bf16" and dim <= 128 and not few and not prompts:
        tile = 256 if tiles(256) * kv >= 4 * cus else 128
    return tile, tiles(tile) * kv < 4 * cus and nseq <= 384 and width * page // 32 > 4


class Many:
    """A case of a few key-value heads, whose heads are repeated up to `kv` of them."""

    def __init__(self, vs, tile, lens, counts, kv, group=1, dim=64, page=32, distinct=3, dtype="bf16", **kw):
        self.c = c = Rows(vs, lens, counts, distinct * group, distinct, dim, page, dtype, **kw)
        self.vs, self.kv, self.group, self.of = vs, kv, group, np.arange(kv) % distinct
        got = kernel(vs, c.nrows, kv * group, kv, len(lens), c.table.shape[1], page, dim, dtype)
        assert got == (tile, False), got
        self.qb = self.wide(c.qb)
        self.mem = vs.DeviceArray(c.pool.shape[:3] + (kv,) + c.pool.shape[4:], dtype)
        self.cache = vs.PagedKVCache(len(c.pool), page, kv, dim, dtype=dtype, memory=self.mem)
        self.fill()

    def wide(self, x):
        """[rows, distinct * group, dim] with its heads repeated."""
        x = x.reshape(len(x), -1, self.group, self.c.dim)[:, self.of]
        return np.ascontiguousarray(x.reshape(len(x), self.kv * self.group, self.c.dim))

    def fill(self):
        self.mem.upload(np.ascontiguousarray(self.c.pool[:, :, :, self.of]))

    def keys_times(self, factor):
        """Every key of position p times factor(p)."""
        c = self.c
        for b, n in enumerate(c.lens):
            kb, k = D.stored(c.k[b] * factor(np.arange(n))[:, None, None], c.dtype)
            D.write_rows(c.pool[:, 0], c.table, b, 0, kb, D.stored(c.v[b], c.dtype)[0], c.page, c.dtype)
            c.k[b] = k.astype(np.float64)
        self.fill()

    def run(self, in_place=False, **kw):
        A, c, heads = self.vs.DeviceArray, self.c, self.kv * self.group
        q, lse = A.of(self.qb, c.dtype), A.of(np.full((c.nrows, heads), 77.0), "f32")
        out = q if in_place else A.of(np.full((c.nrows, heads, c.dim), 0x7FC1 if c.dtype == "bf16" else 77.0), c.dtype)
        self.cache.attend_rows(c.seqs, q, out, lse=lse, starts=A.of(c.starts, "i32"), **kw)
        self.cache.check()
        got = out.numpy().reshape(c.nrows, self.kv, self.group, c.dim), lse.numpy().reshape(c.nrows, self.kv, self.group)
        n = c.kv
        for x in got:  # equal heads have equal answers
            x = x if x.dtype == np.uint16 else x.view(np.uint32)
            assert (x == x[:, self.of]).all()
        o = got[0][:, :n].reshape(c.nrows, n * self.group, c.dim)
        return (D.from_bf16(o) if c.dtype == "bf16" else o), got[1][:, :n].reshape(c.nrows, n * self.group)

    def check(self, missing=lambda b: (), **kw):
        self.c.compare(self.run(**kw), kw.get("window", 0), kw.get("sinks", 0), kw.get("scale"), kw.get("causal", True), missing)


# (rows of a tile, key-value heads, lengths, rows): odd numbers of blocks and even ones, tiles that are not full, rows
# from the first position on and behind others
LARGE = (256, 256, [300, 257, 70], [290, 150, 64])
MIDDLE = (128, 128, [390, 257, 100], [390, 250, 70])
BOTH = pytest.mark.parametrize("tile,kv,lens,counts", [LARGE, MIDDLE], ids=["256", "128"])


@BOTH
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", range(16, 129, 16))
def test_head_dims(vs, tile, kv, lens, counts, dim, causal):
    Many(vs, tile, lens, counts, kv, dim=dim, tail=2).check(causal=causal)


@BOTH
@pytest.mark.parametrize("page", [64, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 4), (33, 33), (64, 0), (100, 40), (31, 300), (2**31 - 1, 2**31 - 1)])
def test_window_and_sinks(vs, tile, kv, lens, counts, page, window, sinks):
    Many(vs, tile, lens, counts, kv, dim=48, page=page, lead=1).check(window=window, sinks=sinks)


@pytest.mark.parametrize("group,tile,kv,rows", [(3, 256, 128, [200, 100, 303]), (5, 256, 256, [90, 7, 31]), (17, 256, 64, [41, 90, 100]),
                                                (130, 256, 64, [9, 2, 20]), (3, 128, 128, [150, 64, 20])])
def test_groups(vs, group, tile, kv, rows):
    """Tiles that end inside a row's heads."""
    Many(vs, tile, [300, 111, 400], rows, kv, group=group, dim=32, distinct=2).check()


@pytest.mark.parametrize("n,tile", [(400, 256), (400, 128)])
def test_many_sequences(vs, n, tile):
    """Tiles are numbered with gaps."""
    rng, kv = np.random.default_rng(n), 4 if tile == 256 else 1
    lens = rng.integers(0, 150, n)
    counts = np.minimum(rng.integers(0, 9, n), lens)
    counts[7] = lens[7] = 129
    Many(vs, tile, lens, counts, kv, group=20, dim=32, distinct=1, tail=3).check()


@BOTH
@pytest.mark.parametrize("causal", [True, False])
def test_scores_that_grow(vs, tile, kv, lens, counts, causal):
    """References are raised in either block of a step, with weights of the first one waiting."""
    m = Many(vs, tile, lens, counts, kv, dim=64, spread=2.0)
    m.keys_times(lambda p: 0.2 + 3.0 * (p // 32 % 2))
    m.check(causal=causal)
    m.keys_times(lambda p: 1.0 + p / 100)
    m.check(causal=causal)
    m.check(scale=-0.3, causal=causal)


@BOTH
@pytest.mark.parametrize("causal", [True, False])
def test_missing_pages(vs, tile, kv, lens, counts, causal):
    """Whichever block of a step is left out."""
    m = Many(vs, tile, lens, counts, kv, dim=32)
    c = m.c
    c.table[0, [1, 4, 5]] = [-1, len(c.pool), -7]
    c.table[1, :8] = -1
    gone = [list(range(32, 64)) + list(range(128, 192)), range(256), []]
    c.sequences(np.zeros(len(c.pool), np.int32))
    m.check(causal=causal, missing=lambda b: gone[b])


@BOTH
@pytest.mark.parametrize("at", [5, 37, 64, 131, 161, 255])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 70])
def test_what_a_row_does_not_see_may_be_anything(vs, tile, kv, lens, counts, at, bad, window):
    """A value that is not finite, in either block of a step: rows that do not see it are as without it."""
    m = Many(vs, tile, lens, counts, kv, dim=32, spread=0.5)
    c, (free, free_lse) = m.c, m.run(window=window)
    _, vp = D.places(32, "bf16")
    c.pool[c.table[0, at // 32], 0, 1, 1, vp[at % 32, 5]] = D.stored(np.full(1, bad), "bf16")[0][0]
    m.fill()
    out, lse = m.run(window=window)
    n, rows = lens[0], counts[0]
    sees = np.zeros(c.nrows, bool)
    sees[:rows] = P.seen_mask(np.arange(n - rows, n), n, window, 0)[:, at]
    assert sees.any()  # (all of them do where the position is before the first row's)
    hit = np.zeros(out.shape, bool)
    hit[sees, 1, 5] = True
    assert np.array_equal(lse, free_lse) and not np.isfinite(out[hit]).any()
    if not np.isnan(bad):  # (no weight of these scores is too small for 32 bits)
        assert (out[hit] == bad).all()
    # blocks without a hidden position go through other instructions, whose sums are in another order
    want = np.where(hit, 0, free)
    np.testing.assert_allclose(np.where(hit, 0, out), want, rtol=0, atol=np.abs(want).max() * 2.0 ** -6)


@BOTH
@pytest.mark.parametrize("at", [37, 161])
def test_keys_that_are_not_finite(vs, tile, kv, lens, counts, at):
    m = Many(vs, tile, lens, counts, kv, dim=64)
    c, free = m.c, m.run()
    kp, _ = D.places(64, "bf16")
    c.pool[c.table[0, at // 32], 0, 0, 0, kp[at % 32, 3]] = D.stored(np.full(1, np.nan), "bf16")[0][0]
    m.fill()
    sees = np.zeros(c.nrows, bool)
    sees[:counts[0]] = np.arange(lens[0] - counts[0], lens[0]) >= at
    for got, want in zip(m.run(), free):
        assert np.array_equal(got[~sees], want[~sees]) and np.array_equal(got[:, 1:], want[:, 1:])
        assert np.isnan(got[sees][:, 0]).all()


@BOTH
def test_in_place_and_rows_before_the_first_position(vs, tile, kv, lens, counts):
    m = Many(vs, tile, lens, counts, kv, dim=32)
    assert np.array_equal(m.run(in_place=True)[0], m.run()[0])
    m.c.lens = np.array([120, 0, -9], np.int32)
    m.c.sequences(np.zeros(len(m.c.pool), np.int32))
    m.check()


@pytest.mark.parametrize("n", [4, 40, 300])
def test_starts_that_do_not_ascend(vs, n):
    """Sequences that name the same rows again and again: more tiles than there is room for are not answered, and the
    next call is as ever."""
    c = Rows(vs, [400] + [150] * (n - 1), [200] + [0] * (n - 1), 4, 2, 32, 32, "bf16")
    assert kernel(vs, 200, 4, 2, n, c.table.shape[1], 32, 32, "bf16")[1]
    want, good = c.run(), c.starts
    c.starts = np.arange(n + 1) % 2 * 200
    out, lse = c.run()
    assert np.isnan(out).all() and (lse == 77.0).all()
    c.starts = good
    for got, w in zip(c.run(), want):
        assert np.array_equal(got, w)


@pytest.mark.parametrize("dtype,dim,counts", [("f32", 64, [90, 33, 70]), ("f32", 192, [90, 33, 70]), ("bf16", 192, [90, 33, 90]),
                                              ("bf16", 64, [20, 1, 3]), ("bf16", 256, [1, 1, 1])])
def test_small_tiles_that_are_not_divided(vs, dtype, dim, counts):
    m = Many(vs, 64, [300, 257, 120], counts, 384, dim=dim, dtype=dtype, distinct=2)
    m.check()
    m.check(window=50, sinks=3)


class Over:
    """A buffer of another shape and type over an array's memory."""

    def __init__(self, base, shape, dtype):
        self.base, self.shape, self.dtype = base, shape, dtype

    def data_ptr(self):
        return self.base.data_ptr()

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))


def test_outputs_over_what_tells_the_places(vs):
    """Starts, lengths and the table are read while rows are answered and stored."""
    A = vs.DeviceArray
    c = Rows(vs, [64, 30], [5, 2], 2, 1, 32, 32, "bf16", width=300)
    rows, starts = c.nrows, A.of(c.starts, "i32")
    q, k, rot = A.of(c.qb, "bf16"), A((rows, 1, 32), "bf16"), vs.Rotary(32)
    for base in (starts, c.seqs.lens, c.seqs.table):
        over = Over(base, (rows, 2, 32), "bf16")
        with pytest.raises(ValueError, match="overlaps starts"):
            c.cache.attend_rows(c.seqs, q, over, starts=starts)
        with pytest.raises(ValueError, match="overlaps starts"):
            c.cache.attend_rows(c.seqs, q, A((rows, 2, 32), "bf16"), lse=Over(base, (rows, 2), "f32"), starts=starts)
        with pytest.raises(ValueError, match="overlaps starts"):
            c.cache.append(c.seqs, k, k, starts=starts, rotary=rot, q=q, q_out=over)
    c.compare(c.run())


@pytest.mark.parametrize("lens,counts", [([150, 90], [9, 20]), ([3000, 90], [9, 20])])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 6])
def test_few_rows_and_values_that_are_not_finite(vs, lens, counts, bad, window):
    """Weights in several parts: a value that is not finite counts once, with the whole weight, where it is seen."""
    c = Rows(vs, lens, counts, 4, 2, 64, 32, "bf16", spread=0.5)
    assert kernel(vs, c.nrows, 4, 2, 2, c.table.shape[1], 32, 64, "bf16")[0] == 64 and c.nrows * 2 <= 2 * 64
    free, n, at = c.run(window=window), lens[0], lens[0] - 6
    _, vp = D.places(64, "bf16")
    c.pool[c.table[0, at // 32], 0, 1, 1, vp[at % 32, 5]] = D.stored(np.full(1, bad), "bf16")[0][0]
    c.mem.upload(c.pool)
    out, lse = c.run(window=window)
    hit = np.zeros(out.shape, bool)
    hit[:counts[0], 2:, 5] = P.seen_mask(np.arange(n - counts[0], n), n, window, 0)[:, at, None]
    assert hit.any() and not hit[:counts[0], 2:, 5].all()
    assert np.array_equal(lse, free[1]) and not np.isfinite(out[hit]).any()
    if not np.isnan(bad):  # (no weight of these scores is too small for 32 bits)
        assert (out[hit] == bad).all()
    want = np.where(hit, 0, free[0])
    np.testing.assert_allclose(np.where(hit, 0, out), want, rtol=0, atol=np.abs(want).max() * 2.0 ** -7)


@pytest.mark.parametrize("dtype,dim,kv,counts", [("f32", 256, 2, [90, 40]), ("bf16", 256, 2, [90, 40]), ("bf16", 128, 256, [500, 600])])
def test_recorded_calls(vs, dtype, dim, kv, counts):
    """Kernels of more shared memory than a launch has by itself, recorded and replayed with other work between."""
    A, st = vs.DeviceArray, Stream()
    c = Rows(vs, [700, 650], counts, kv, kv, dim, 32, dtype)
    want = c.run()
    q, starts, (out, lse) = A.of(c.qb, dtype), A.of(c.starts, "i32"), c.poisoned()
    c.cache.attend_rows(c.seqs, q, out, lse=lse, starts=starts, stream=st.ptr)  # (scratch of this stream)
    st.sync()
    st.begin()
    c.cache.attend_rows(c.seqs, q, out, lse=lse, starts=starts, stream=st.ptr)
    graph = st.end()
    for _ in range(3):
        out.upload(c.poisoned()[0].numpy())
        other = c.run()
        st.replay(graph)
        for got in (c.values(out, lse), other):
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
