"""Where the rows of a batch go, against the rule row by row."""
import numpy as np
import pytest

import _prompt as P
from _hip import Stream

pytestmark = pytest.mark.gpu


def setup(vs, counts, lens, page=32, width=None, seed=0, npages=500):
    A, rng = vs.DeviceArray, np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    width = width or max(1, -(-int(max(lens, default=1)) // page))
    table = rng.integers(-1, npages + 2, (len(lens), width)).astype(np.int32)  # (missing ones and ones past the cache among them)
    cache = vs.PagedKVCache(npages, page, 1, 16)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of(lens, "i32"), A.of(np.zeros(npages), "i32"))
    return cache, seqs, table


def run(vs, cache, seqs, counts, nrows, stream=0):
    A = vs.DeviceArray
    outs = [A.of(np.full(seqs.n + 1, 77), "i32")] + [A.of(np.full(nrows, 77), "i32") for _ in range(3)]
    cache.rows(seqs, counts if isinstance(counts, int) else A.of(counts, "i32"), outs[0], sequence=outs[1], position=outs[2],
               slot=outs[3], stream=stream)
    return outs


def compare(outs, want):
    for got, w in zip(outs, want):
        assert np.array_equal(got.numpy(), w)


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 1023, 1024, 1025, 3000, 8191, 8192, 8193, 20000])
@pytest.mark.parametrize("most", [1, 9])
def test_sequences(vs, n, most):
    rng = np.random.default_rng(n)
    lens, counts = rng.integers(0, 300, n), rng.integers(-1, most + 1, n)
    cache, seqs, table = setup(vs, counts, lens, seed=n)
    total = int(np.maximum(counts, 0).sum())
    for nrows in {total, total + 100}:
        outs = run(vs, cache, seqs, counts, nrows)
        compare(outs, P.rows_of(counts, lens, table, 32, 500, nrows))
    cache.check()
    cache.close()


@pytest.mark.parametrize("page", [32, 128, 1024])
def test_long_counts_and_narrow_tables(vs, page):
    lens, counts = [5000, 70, 10, 0, 3000], [4000, 70, 20, 3, 1]
    cache, seqs, table = setup(vs, counts, lens, page, width=2)
    outs = run(vs, cache, seqs, counts, 4094 + 3)
    compare(outs, P.rows_of(counts, lens, table, page, 500, 4097))
    cache.check()


def test_one_count_for_all(vs):
    cache, seqs, table = setup(vs, None, [40, 9, 300])
    compare(run(vs, cache, seqs, 4, 12), P.rows_of([4] * 3, [40, 9, 300], table, 32, 500, 12))
    compare(run(vs, cache, seqs, 0, 2), P.rows_of([0] * 3, [40, 9, 300], table, 32, 500, 2))


@pytest.mark.parametrize("n", [3, 9000])
def test_more_rows_than_there_are(vs, n):
    """Rows past nrows are left out, and the check says so; starts past 2^31 - 1 stay there."""
    counts = np.full(n, 5)
    cache, seqs, table = setup(vs, counts, np.full(n, 100))
    compare(run(vs, cache, seqs, counts, 5 * n - 3), P.rows_of(counts, np.full(n, 100), table, 32, 500, 5 * n - 3))
    with pytest.raises(ValueError, match="more rows"):
        cache.check()
    cache.check()
    counts[:3] = 2**31 - 1
    starts = run(vs, cache, seqs, counts, 40)[0].numpy()
    assert np.array_equal(starts, np.minimum(np.concatenate([[0], counts.astype(np.int64).cumsum()]), 2**31 - 1))
    with pytest.raises(ValueError, match="more rows"):
        cache.check()


def test_single_outputs_and_starts_alone(vs):
    A = vs.DeviceArray
    counts, lens = [3, 0, 5], [40, 9, 300]
    cache, seqs, table = setup(vs, counts, lens)
    want = P.rows_of(counts, lens, table, 32, 500, 8)
    for i, name in enumerate(("sequence", "position", "slot")):
        starts, out = A((4,), "i32"), A((8,), "i32")
        cache.rows(seqs, A.of(counts, "i32"), starts, **{name: out})
        assert np.array_equal(out.numpy(), want[i + 1]) and np.array_equal(starts.numpy(), want[0])
    starts = A((4,), "i32")
    cache.rows(seqs, A.of(counts, "i32"), starts)
    assert np.array_equal(starts.numpy(), want[0])
    cache.check()


def test_streams_and_graphs(vs):
    A = vs.DeviceArray
    counts, lens = [3, 0, 5], [40, 9, 300]
    cache, seqs, table = setup(vs, counts, lens)
    st, c, outs = Stream(), A.of(counts, "i32"), [A((4,), "i32")] + [A((8,), "i32") for _ in range(3)]
    st.begin()
    cache.rows(seqs, c, outs[0], sequence=outs[1], position=outs[2], slot=outs[3], stream=st.ptr)
    graph = st.end()
    for counts in ([3, 0, 5], [1, 6, 1], [8, 0, 0]):
        c.upload(np.array(counts))
        st.replay(graph)
        compare(outs, P.rows_of(counts, lens, table, 32, 500, 8))


def test_refusals(vs):
    A = vs.DeviceArray
    cache, seqs, _ = setup(vs, None, [40, 9, 300])
    counts, starts, out = A.of([1, 2, 3], "i32"), A((4,), "i32"), A((6,), "i32")
    for args, kw in (((-1, starts), {}), ((2**31, starts), {}), ((A((2,), "i32"), starts), {}), ((counts, A((3,), "i32")), {}),
                     ((counts, starts), dict(sequence=out, position=A((5,), "i32"))), ((counts, starts), dict(slot=out, position=out)),
                     ((counts, starts), dict(slot=A((6,), "f32"))), ((counts, starts), dict(sequence=seqs.lens)),
                     ((out, out), {})):
        with pytest.raises(ValueError):
            cache.rows(seqs, *args, **kw)


@pytest.mark.parametrize("n", [3, 9000])
def test_starts_alone_take_no_time_for_rows(vs, n):
    """nrows is 2^31 - 1 where no row's place is asked for: none of them is visited (doing so takes half a second)."""
    import time

    A = vs.DeviceArray
    counts = np.arange(n) % 7
    cache, seqs, _ = setup(vs, counts, np.full(n, 40))
    starts, c = A((n + 1,), "i32"), A.of(counts, "i32")
    cache.rows(seqs, c, starts)
    cache.check()
    t = time.perf_counter()
    for _ in range(10):
        cache.rows(seqs, c, starts)
    cache.check()
    assert time.perf_counter() - t < 0.5
    assert np.array_equal(starts.numpy(), np.concatenate([[0], counts.cumsum()]))


def test_no_slots_behind_an_extend_that_did_not_fit(vs):
    """The sequences' last positions hold tokens in use then: who stores by the slots leaves them alone, as append does.
    Other sequences' rows, and everyone's behind the check, have theirs."""
    A = vs.DeviceArray
    cache = vs.PagedKVCache(5, 32, 1, 16)
    seqs = cache.new_sequences(2, 8)
    cache.extend(seqs, A.of([90, 10], "i32"))
    cache.check()
    other = vs.KVSequences(A.of(np.full((1, 8), -1), "i32"), A.of([0], "i32"), seqs.refs)
    cache.extend(other, 5)
    cache.check()
    table, lens = seqs.table.numpy(), [90, 10]
    cache.extend(seqs, A.of([70, 0], "i32"))  # (not a page is left)
    counts = [40, 3]
    want = P.rows_of(counts, lens, table, 32, 5, 45)
    closed = [w.copy() for w in want]
    closed[3][:40] = -1
    compare(run(vs, cache, seqs, counts, 45), closed)
    compare(run(vs, cache, other, [5], 5), P.rows_of([5], [5], other.table.numpy(), 32, 5, 5))
    with pytest.raises(vs.VsError, match="pages short"):
        cache.check()
    compare(run(vs, cache, seqs, counts, 45), want)


@pytest.mark.parametrize("n", [3, 9000])
def test_more_rows_than_one_pass_of_the_grid(vs, n):
    """Past 512 workgroups of 1,024 rows each."""
    counts = np.full(n, 700_000 // n)
    lens = counts + np.arange(n) % 50
    cache, seqs, table = setup(vs, counts, lens, width=20, npages=400)
    nrows = int(counts.sum()) + 9
    starts = np.concatenate([[0], counts.cumsum()])
    b = np.repeat(np.arange(n), counts)
    pos = lens[b] - (starts[b + 1] - np.arange(len(b)))
    page = np.where(pos < 20 * 32, table[b, np.minimum(pos // 32, 19)], -1)
    slot = np.where((page >= 0) & (page < 400), page * 32 + pos % 32, -1)
    pad = lambda x: np.concatenate([x, np.full(9, -1)])  # noqa: E731
    compare(run(vs, cache, seqs, counts, nrows), [starts, pad(b), pad(pos), pad(slot)])
    cache.check()
