"""Refusals of the decoding entry points that need no GPU, and the plain forms' own checks."""
import ctypes

import numpy as np
import pytest

import _decode as D

INVALID, UNSUPPORTED = 1, 4


@pytest.fixture(scope="module")
def lib():
    from vector_store import _native

    return _native.load()


@pytest.mark.parametrize("args,code,word", [
    ((0, 0, 32, 1, 1, 64, 1), INVALID, "npages"),
    ((0, 4, 32, 0, 1, 64, 1), INVALID, "layers"),
    ((0, 4, 32, 1, -1, 64, 1), INVALID, "kv_heads"),
    ((0, 4, 16, 1, 1, 64, 1), INVALID, "page_size"),
    ((0, 4, 48, 1, 1, 64, 1), INVALID, "page_size"),
    ((0, 4, 2048, 1, 1, 64, 1), INVALID, "page_size"),
    ((0, 4, 32, 1, 1, 0, 1), UNSUPPORTED, "head_dim"),
    ((0, 4, 32, 1, 1, 72, 1), UNSUPPORTED, "head_dim"),
    ((0, 4, 32, 1, 1, 272, 1), UNSUPPORTED, "head_dim"),
    ((0, 4, 32, 1, 1, 64, 2), INVALID, "dtype"),
    ((0, 1 << 31, 32, 1, 1, 64, 1), UNSUPPORTED, "pages"),
])
def test_cache_refusals(lib, args, code, word):
    h = ctypes.c_void_p(5)
    assert lib.vs_kv_create(*args, None, ctypes.byref(h)) == code
    assert word in lib.vs_last_error().decode() and not h.value


def test_unaligned_memory_and_null_handles(lib):
    h = ctypes.c_void_p()
    assert lib.vs_kv_create(0, 4, 32, 1, 1, 64, 1, ctypes.c_void_p(24), ctypes.byref(h)) == INVALID
    assert lib.vs_kv_create(0, 4, 32, 1, 1, 64, 1, None, None) == INVALID
    z = ctypes.c_void_p()
    assert lib.vs_kv_attend(z, z, 0, 1, z, 0, 0, z, 0, 0, z, 0, 0, z, 0, 0, z, 1.0, 0, 0, z) == INVALID
    assert lib.vs_kv_append(z, z, 0, z, 0, 0, z, 0, 0, z, 0, z) == INVALID
    assert lib.vs_kv_read(z, z, 0, 0, 0, 0, z, z, z) == INVALID
    assert lib.vs_kv_extend(z, z, 1, z, z) == INVALID
    assert lib.vs_kv_fork(z, z, z, z, z) == INVALID
    assert lib.vs_kv_free(z, z, z, 0, z) == INVALID
    assert lib.vs_kv_evict(z, z, 1, 0, z) == INVALID
    assert lib.vs_kv_compact(z, z, z, z) == INVALID
    assert lib.vs_kv_copy(z, z, z, 0, z) == INVALID
    assert lib.vs_kv_check(z, z) == INVALID
    assert lib.vs_beam_select(z, z, 0, 1, 1, 1, 1, z, z, 0, 1, z, z, z, z, z) == INVALID
    assert lib.vs_beam_reorder(z, z, 0, z, 0, 0, z, 0, 0, z, z) == INVALID
    lib.vs_kv_destroy(z)
    lib.vs_beam_destroy(z)


class Fake:
    def __init__(self, shape, dtype="f32", stride=None):
        self.shape, self.dtype = shape, dtype
        n, st = 1, []
        for s in reversed(shape):
            st.append(n)
            n *= s
        self._st = stride or tuple(reversed(st))

    def data_ptr(self):
        return 4096

    def stride(self):
        return self._st


def test_buffers_are_checked_before_any_call():
    import vector_store as vs

    good = dict(table=Fake((3, 2), "i32"), lens=Fake((3,), "i32"), refs=Fake((4,), "i32"))
    vs.KVSequences(**good)
    for name, bad in [("table", Fake((3, 2), "f32")), ("table", Fake((6,), "i32")), ("lens", Fake((4,), "i32")),
                      ("lens", Fake((3,), "i32", (2,))), ("table", Fake((3, 2), "i32", (4, 1))),
                      ("refs", Fake((4,), "torch.int64"))]:
        with pytest.raises(ValueError):
            vs.KVSequences(**{**good, name: bad})


def test_rows_views():
    from vector_store import decode

    p, st = decode._rows(Fake((2, 3, 16), "torch.bfloat16", (100, 16, 1)), "q", (2, 3, 16), 1)
    assert p == 4096 and st == (100, 16, 1)
    for bad in (Fake((2, 3, 16), "bf16", (1, 2, 6)), Fake((2, 3, 16), "f32"), Fake((2, 3, 32), "bf16")):
        with pytest.raises(ValueError):
            decode._rows(bad, "q", (2, 3, 16), 1)


def test_places_cover_a_block():
    for dtype in ("bf16", "f32"):
        for dim in (16, 48, 80, 256):
            for p in D.places(dim, dtype):
                assert sorted(p.ravel()) == list(range(32 * dim))


def test_plain_attention_masks():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((4, 8)), rng.standard_normal((20, 2, 8)), rng.standard_normal((20, 2, 8))
    assert list(D.visible(20, 3, 2)) == [0, 1, 17, 18, 19] and list(D.visible(2, 5, 9)) == [0, 1]
    out, lse = D.attend(q, k, v, D.visible(20, 1, 0), 1.0)
    np.testing.assert_allclose(out, np.repeat(v[19], 2, axis=0))
    np.testing.assert_allclose(lse, np.einsum("hd,hd->h", q, np.repeat(k[19], 2, axis=0)))


def test_pages_model():
    """Two beams on one partly filled page: the first keeps it, the second takes a copy; then both own theirs."""
    m = D.Pages([[0, -1], [0, -1]], [5, 5], [2, 0, 0], 32)
    assert m.extend(1) is None and m.table.tolist() == [[0, -1], [1, -1]]
    assert m.refs.tolist() == [1, 1, 0] and m.copies == [(0, 1)]
    assert m.extend(27) == "pages" and m.lens.tolist() == [6, 6]
    f = m.fork([1, 1])
    assert f.refs.tolist() == [0, 2, 0]
    c = f.compact()
    assert c.table[0, 0] == 0 and c.refs.tolist() == [2, 0, 0]


def test_beam_model_order():
    x = np.array([[1.0, 1.0, 0.0], [1.0, 1.0, 0.0]])
    s, t, p, f = D.beam_select(x, np.zeros((1, 2)), np.zeros((1, 2)), 1, 5)
    assert t.tolist() == [[0, 1, 0, 1, 2]] and p.tolist() == [[0, 0, 1, 1, 0]] and f.tolist() == [[0, 1, 0, 1, 0]]
