"""Extends by very many pages at once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_more_than_a_million_pages_for_one_sequence(vs):
    """Given where they are there, refused where they are not: by the pages alone, however many one sequence takes."""
    A, npages = vs.DeviceArray, (1 << 20) + 100
    cache = vs.PagedKVCache(npages, 32, 1, 16)
    refs = np.zeros(npages, np.int32)
    refs[[3, 70_000]] = 1
    table = np.full((2, npages), -1, np.int32)
    seqs = vs.KVSequences(A.of(table, "i32"), A.of([0, 0], "i32"), A.of(refs, "i32"))
    counts = np.array([((1 << 20) + 50) * 32 - 7, 70])
    cache.extend(seqs, A.of(counts + [0, 32 * 50], "i32"))
    with pytest.raises(vs.VsError, match="5 pages short"):
        cache.check()
    cache.extend(seqs, A.of(counts, "i32"))
    cache.check()
    free, first = np.flatnonzero(refs == 0), (1 << 20) + 50
    table[0, :first], table[1, :3] = free[:first], free[first:first + 3]
    refs[free[:first + 3]] = 1
    assert np.array_equal(seqs.table.numpy(), table) and np.array_equal(seqs.lens.numpy(), counts)
    assert np.array_equal(seqs.refs.numpy(), refs)
    cache.close()


@pytest.mark.parametrize("n", [3, 40, 1024, 1500])
def test_sums_past_32_bits_are_refused(vs, n):
    """Each of n sequences asks for 2^26 pages, by which a sum of 32 bits would come to 0 at 64 of them."""
    A = vs.DeviceArray
    cache = vs.PagedKVCache(50, 32, 1, 16)
    # (rows are not read where nothing is held, and not written where the plan is refused: one row stands for all)
    width = (2**31 - 1) // 32

    class Wide:
        def __init__(self, base):
            self.base, self.shape, self.dtype = base, (n, width), base.dtype

        def data_ptr(self):
            return self.base.data_ptr()

        def stride(self):
            return (width, 1)

    lens = np.zeros(n, np.int32)
    seqs = vs.KVSequences(Wide(A.of([[-1]], "i32")), A.of(lens, "i32"), A.of(np.zeros(50), "i32"))
    cache.extend(seqs, width * 32)
    with pytest.raises(vs.VsError, match=f" {min(n * width - 50, 2**31 - 1)} pages short"):
        cache.check()
    assert not seqs.lens.numpy().any() and not seqs.refs.numpy().any()
    cache.close()
