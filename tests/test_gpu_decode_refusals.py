"""Arguments that the decoding calls have to refuse on the host: nothing is launched for them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Shifted:
    """A buffer whose address is some bytes further on."""

    def __init__(self, base, by):
        self.base, self.by, self.shape, self.dtype = base, by, base.shape, base.dtype

    def data_ptr(self):
        return self.base.data_ptr() + self.by

    def stride(self):
        return self.base.stride()


@pytest.mark.parametrize("which", ["table", "lens", "refs"])
@pytest.mark.parametrize("by", [1, 2])
def test_sequences_off_their_alignment(vs, which, by):
    """An atomic on a misaligned count would fault."""
    A = vs.DeviceArray
    cache = vs.PagedKVCache(4, 32, 1, 16)
    parts = dict(table=A.of([[0, 1], [2, -1]], "i32"), lens=A.of([33, 5], "i32"), refs=A.of([1, 1, 1, 0], "i32"))
    good = vs.KVSequences(**parts)
    bad = vs.KVSequences(**{**parts, which: Shifted(parts[which], by)})
    q, k = A((2, 1, 16), "bf16"), A((2, 1, 16), "bf16")
    out = vs.KVSequences(A((2, 2), "i32"), A((2,), "i32"), parts["refs"])
    for f in (lambda: cache.attend(bad, q, k), lambda: cache.append(bad, k, k), lambda: cache.extend(bad, 1),
              lambda: cache.fork(bad, A.of([0, 1], "i32"), out), lambda: cache.fork(good, A.of([0, 1], "i32"), bad),
              lambda: cache.free(bad), lambda: cache.evict(bad, 4), lambda: cache.compact(bad), lambda: cache.compact(good, bad),
              lambda: cache.read(bad, 0, 0, k, k), lambda: cache.compact(good, others=[bad])):
        with pytest.raises(ValueError, match="aligned|shape|counts|another table"):
            f()
    cache.check()
    assert parts["lens"].numpy().tolist() == [33, 5] and parts["refs"].numpy().tolist() == [1, 1, 1, 0]
    assert np.array_equal(parts["table"].numpy(), [[0, 1], [2, -1]])
    cache.close()
