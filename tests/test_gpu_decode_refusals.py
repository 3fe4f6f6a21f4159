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


def test_a_selection_over_its_own_inputs(vs):
    """In place with as many candidates as beams; refused where one request's outputs would lie on another's scores."""
    A, rng = vs.DeviceArray, np.random.default_rng(1)
    R, W, V = 40, 4, 3001
    x, sc = rng.standard_normal((R * W, V)), -5 * rng.random((R, W)).astype(np.float32)
    fin = (rng.random((R, W)) < 0.2).astype(np.uint8)
    lg, bs = A.of(x, "f32"), vs.BeamSearch()
    so, fo, to, po = A((R, W), "f32"), A((R, W), "u8"), A((R, W), "i32"), A((R, W), "i32")
    bs.select(lg, A.of(sc, "f32"), so, to, po, finished=A.of(fin, "u8"), finished_out=fo, eos=2)
    s, f = A.of(sc, "f32"), A.of(fin, "u8")
    t2, p2 = A((R, W), "i32"), A((R, W), "i32")
    bs.select(lg, s, s, t2, p2, finished=f, finished_out=f, eos=2)
    for a, b in ((s, so), (f, fo), (t2, to), (p2, po)):
        assert np.array_equal(a.numpy(), b.numpy())

    class Part(Shifted):
        def __init__(self, base, shape, by=0):
            super().__init__(base, by)
            self.shape = shape

        def stride(self):
            return (self.shape[1], 1)

    out = lambda k: (A((R, k), "f32"), A((R, k), "i32"), A((R, k), "i32"))  # noqa: E731
    s, f = A.of(sc, "f32"), A.of(fin, "u8")
    so, to, po = out(2)
    for args, kw in (((s, Part(s, (R, 2)), to, po), {}), ((s, so, to, po), dict(finished=f, finished_out=Part(f, (R, 2)))),
                     ((s, Part(s, (R, 2), 8), to, po), {})):
        with pytest.raises(ValueError, match="overlaps"):
            bs.select(lg, *args, **kw)
    half = Part(s, (R // 2, W)), Part(s, (R // 2, W), R // 2 * W * 4)
    one = A((R // 2, W), "i32"), A((R // 2, W), "i32")
    bs.select(Part(lg, (R // 2 * W, V)), half[0], half[1], *one)  # (side by side in one buffer)
    with pytest.raises(ValueError, match="overlaps"):
        bs.select(Part(lg, (R // 2 * W, V)), half[0], Part(s, (R // 2, W), R // 2 * W * 4 - 4), *one)
    bs.close()


class Cut(Shifted):
    """Some rows of a buffer, at an offset in bytes."""

    def __init__(self, base, shape, by=0):
        super().__init__(base, by)
        self.shape = shape

    def stride(self):
        return (self.shape[1], 1) if len(self.shape) == 2 else (1,)


def test_sequences_that_overlap_in_part(vs):
    """Rows that one workgroup writes while another reads them."""
    A = vs.DeviceArray
    cache = vs.PagedKVCache(4, 32, 1, 16)
    table, lens, refs = A.of(np.full((4, 2), -1), "i32"), A.of(np.zeros(4), "i32"), A.of(np.zeros(8), "i32")
    seqs = lambda t=0, ln=0, r=0: vs.KVSequences(Cut(table, (2, 2), t), Cut(lens, (2,), ln), Cut(refs, (4,), r))  # noqa: E731
    parents = A.of([0, 1], "i32")
    for out in (seqs(8, 8), seqs(16, 4), seqs(16, 8, 4)):
        with pytest.raises(ValueError, match="fork"):
            cache.fork(seqs(), parents, out)
    for bad in (Cut(table, (2,), 24), Cut(lens, (2,), 8)):
        with pytest.raises(ValueError, match="parents lie"):
            cache.fork(seqs(), bad, seqs(16, 8))
    for out in (seqs(8), seqs(0, 4), seqs(0, 0, 8)):
        with pytest.raises(ValueError, match="in part"):
            cache.compact(seqs(), out)
    with pytest.raises(ValueError, match="twice"):
        cache.compact(seqs(), others=[seqs(8)])
    cache.fork(seqs(), parents, seqs(16, 8))  # side by side
    cache.compact(seqs(), seqs(16, 8))
    cache.compact(seqs(), others=[seqs(16)])
    cache.check()
    bs, h, t = vs.BeamSearch(), A.of(np.arange(24).reshape(6, 4), "i32"), A.of([7, 8], "i32")
    state, low = Cut(h, (2, 4)), Cut(h, (2, 4), 64)
    for args, kw in (((Cut(h, (2,), 80), state, low), {}), ((parents, state, low), dict(tail=Cut(h, (2,), 64)))):
        with pytest.raises(ValueError, match="parents or tail"):
            bs.reorder(*args, **kw)
    bs.reorder(Cut(h, (2,)), A((2, 4), "i32"), low, tail=t)
    bs.close()
    cache.close()


def test_more_workgroups_than_a_launch_has(vs):
    """Refused on the host, before the first of a call's kernels (buffers named larger than they are: nothing reads them)."""
    A = vs.DeviceArray
    bs, n = vs.BeamSearch(), 1 << 23
    some = {t: A((16,), t) for t in ("f32", "i32", "bf16")}
    with pytest.raises(NotImplementedError, match="requests"):
        bs.select(Cut(some["f32"], (n, 5)), Cut(some["f32"], (n, 1)), Cut(A((16,), "f32"), (n, 1), 1 << 40),
                  Cut(some["i32"], (n, 1), 1 << 41), Cut(some["i32"], (n, 1), 1 << 42))
    bs.close()
    cache, n = vs.PagedKVCache(2, 32, 64, 16), 1 << 20
    seqs = vs.KVSequences(Cut(some["i32"], (n, 40)), Cut(some["i32"], (n,)), A.of([0, 0], "i32"))

    class Rows(Cut):
        def stride(self):
            return (64 * 16, 16, 1)

    q = Rows(some["bf16"], (n, 64, 16))
    with pytest.raises(NotImplementedError, match="sequences"):
        cache.attend(seqs, q, q)
    cache.check()
    cache.close()


def test_sequences_whose_join_would_be_no_launch(vs):
    """2^18 sequences of 64 heads in tables that would be split: answered by a workgroup each."""
    A, n, heads, dim, width = vs.DeviceArray, 1 << 18, 64, 16, 40
    cache = vs.PagedKVCache(2, 32, 1, dim)
    one = vs.KVSequences(A.of([[0, 1]], "i32"), A.of([64], "i32"), A.of([1, 1], "i32"))
    ones = A.of(np.full((64, 1, dim), 0x3F80), "bf16")
    cache.append(one, ones, ones, starts=A.of([0, 64], "i32"))
    lens = np.arange(n) % 65
    table = np.full((n, width), -1, np.int32)
    table[:, :2] = [1, 0]
    seqs = vs.KVSequences(A.of(table, "i32"), A.of(lens, "i32"), A.of([1, 1], "i32"))
    q, out = A.of(np.zeros((n, heads, dim), np.uint16), "bf16"), A((n, heads, dim), "bf16")
    lse = A((n, heads), "f32")
    cache.attend(seqs, q, out, lse=lse)
    cache.check()
    assert np.array_equal(out.numpy(), np.broadcast_to(np.where(lens, 0x3F80, 0)[:, None, None], (n, heads, dim)))
    with np.errstate(divide="ignore"):
        want = np.log(lens)[:, None]
    got = lse.numpy()
    assert (got[lens == 0] == -np.inf).all()
    np.testing.assert_allclose(got[lens > 0], np.broadcast_to(want[lens > 0], (int((lens > 0).sum()), heads)), rtol=0,
                               atol=68 * 2.0 ** -23 + 2.0 ** -21 * 25)
    cache.close()


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), 3e38, -2.5e38])
def test_a_scale_that_is_infinite_in_base_two(vs, scale):
    """Scores of 0 times it would be NaN."""
    A, cache = vs.DeviceArray, vs.PagedKVCache(1, 32, 1, 16)
    seqs, q = vs.KVSequences(A.of([[0]], "i32"), A.of([2], "i32"), A.of([1], "i32")), A.of(np.zeros((1, 1, 16)), "bf16")
    out, ones = A((1, 1, 16), "bf16"), A.of(np.full((2, 1, 16), 0x3F80), "bf16")
    cache.append(seqs, ones, ones, starts=A.of([0, 2], "i32"))
    with pytest.raises(ValueError, match="scale"):
        cache.attend(seqs, q, out, scale=scale)
    cache.attend(seqs, q, out, scale=2.3e38)
    assert (out.numpy() == 0x3F80).all()
    cache.close()
