"""Beam search's selection and reordering against their definition in 64 bits."""
import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu

INF = np.inf


class View:
    def __init__(self, base, shape, stride, offset):
        self.base, self.shape, self._stride, self.offset, self.dtype = base, shape, stride, offset, base.dtype

    def data_ptr(self):
        return self.base.data_ptr() + self.offset * (2 if self.dtype == "bf16" else 4)

    def stride(self):
        return self._stride


def select(vs, x, scores, k, dtype="f32", finished=None, eos=-1, pad=0, shift=0):
    A = vs.DeviceArray
    R, W = scores.shape
    rows, V = x.shape
    raw, val = D.stored(x, dtype)
    flat = np.full(shift + rows * (V + pad), D.stored(np.array([np.nan]), dtype)[0][0], raw.dtype)
    for r in range(rows):
        flat[shift + r * (V + pad):][:V] = raw[r]
    lg = View(A.of(flat, dtype), (rows, V), (V + pad, 1), shift)
    so, to, po = A.of(np.full((R, k), 7), "f32"), A.of(np.full((R, k), 7), "i32"), A.of(np.full((R, k), 7), "i32")
    fo = A.of(np.full((R, k), 7), "u8")
    bs = vs.BeamSearch()
    bs.select(lg, A.of(scores, "f32"), so, to, po, finished=None if finished is None else A.of(finished, "u8"),
              finished_out=fo, eos=eos)
    got = so.numpy(), to.numpy(), po.numpy(), fo.numpy()
    bs.close()
    return got, val


def check(got, val, scores, k, finished=None, eos=-1):
    fin = np.zeros(scores.shape, np.uint8) if finished is None else finished
    es, et, ep, ef = D.beam_select(val, scores, fin, eos, k)
    s, t, p, f = got
    assert np.array_equal(np.isfinite(s), np.isfinite(es))
    # log sum exp: exponentials off by 2^-21 with their arguments' rounding, sums of 32 terms and of
    # 64 lanes in 32 bits (38 roundings, 2^-18.7 at most), the rest in 64 bits: below 2^-18 in all.
    # Then the score's own rounding.
    fine = np.isfinite(es)
    np.testing.assert_allclose(s[fine], es[fine], rtol=2.0 ** -23, atol=2.0 ** -18)
    # places may only differ where scores are within that
    same = (t == et) & (p == ep)
    if not same.all():
        for r, i in zip(*np.nonzero(~same)):
            near = np.abs(es[r] - es[r, i]) < 2.0 ** -17 + 2.0 ** -22 * abs(es[r, i])
            assert near.sum() > 1 or i == es.shape[1] - 1, (r, i)
        assert (~same).mean() < 0.02
    assert np.array_equal(f[same], ef[same])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 2047, 2048, 2049, 8191, 50_001])
def test_vocabularies(vs, dtype, V):
    rng = np.random.default_rng(V)
    x, sc = 3 * rng.standard_normal((6, V)), -10 * rng.random((2, 3)).astype(np.float32)
    got, val = select(vs, x, sc, 5, dtype, pad=V % 3, shift=V % 4)
    check(got, val, sc, 5)


@pytest.mark.parametrize("W,k", [(1, 1), (1, 64), (4, 8), (8, 8), (16, 32), (64, 64), (128, 3), (128, 64)])
def test_beams_and_k(vs, W, k):
    rng = np.random.default_rng(W * k)
    x, sc = 2 * rng.standard_normal((3 * W, 5003)), -5 * rng.random((3, W)).astype(np.float32)
    got, val = select(vs, x, sc, k)
    check(got, val, sc, k)


@pytest.mark.parametrize("W,k,V", [(16, 32, 30_000), (64, 64, 9000), (40, 20, 50_000)])
@pytest.mark.parametrize("spread", [0.01, 3.0, 28.0])
def test_scores_near_and_far_apart(vs, W, k, V, spread):
    """One beam's pieces outdo every other beam's best: more candidates than the merge has room for."""
    rng = np.random.default_rng(W)
    x, sc = 2.5 * rng.standard_normal((2 * W, V)), -spread * rng.random((2, W)).astype(np.float32)
    fin = (rng.random((2, W)) < 0.3).astype(np.uint8)
    got, val = select(vs, x, sc, k, "bf16", finished=fin, eos=2)
    check(got, val, sc, k, fin, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ties", [False, True])
def test_large_calls(vs, dtype, ties):
    """Logits enough for the pieces of large calls; with ties, a sixth of every piece is its largest value."""
    rng = np.random.default_rng(17)
    x = rng.standard_normal((32, 530_001)).astype(np.float32)
    if ties:
        x = np.minimum(x, 1)
        x[:, ::3] = np.minimum(x[:, ::3], 0.5)
    sc = -3 * rng.random((4, 8)).astype(np.float32)
    fin = np.zeros((4, 8), np.uint8)
    fin[1, 3] = fin[2, 0] = 1
    got, val = select(vs, x, sc, 20, dtype, finished=fin, eos=530_000, pad=1, shift=1)
    check(got, val, sc, 20, fin, 530_000)


@pytest.mark.parametrize("spread", [0.01, 20.0])
def test_large_calls_of_many_candidates(vs, spread):
    """64 beams and candidates: thresholds over four waves together, and more lists than the merge's registers."""
    rng = np.random.default_rng(64)
    x = 2 * rng.standard_normal((128, 140_001)).astype(np.float32)
    x[5, 140_000] = 90.0  # far above its piece's other logits, and alone in the last one
    sc = -spread * rng.random((2, 64)).astype(np.float32)
    got, val = select(vs, x, sc, 64, "bf16")
    check(got, val, sc, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_exact_ties(vs, dtype):
    """Few distinct logits, so that most of the choice is among equals: in one beam by token, between beams of
    equal rows and scores by beam, wherever the rows start in memory."""
    rng = np.random.default_rng(0)
    V = 6001
    for row in (np.zeros(V), rng.integers(0, 3, V).astype(float), np.where(np.arange(V) % 300 == 7, 5.0, -1.0)):
        x = np.tile(row, (8, 1))
        sc = np.full((2, 4), -3.0, np.float32)
        for k in (1, 5, 64):
            got, val = select(vs, x, sc, k, dtype)
            es, et, ep, _ = D.beam_select(val, sc, np.zeros((2, 4)), -1, k)
            assert np.array_equal(got[1], et) and np.array_equal(got[2], ep)


@pytest.mark.parametrize("k", [3, 64])
def test_more_ties_than_any_list_holds(vs, k):
    """128 equal beams of constant logits: every piece's whole list ties."""
    x, sc = np.full((128, 30_000), 1.25), np.full((1, 128), -1.0, np.float32)
    got, _ = select(vs, x, sc, k)
    assert np.array_equal(got[1][0], np.arange(k)) and not got[2].any()


def test_masked_logits_and_dead_beams(vs):
    """-inf logits, a row of nothing else, -inf and NaN scores, rows with a NaN or +inf; too few candidates."""
    rng = np.random.default_rng(2)
    V = 3000
    x = rng.standard_normal((10, V))
    x[0, 10:] = -INF
    x[1] = -INF
    x[4, 17] = np.nan
    x[5, 2999] = INF
    x[6] = np.nan
    x[7, 1:] = -INF
    sc = np.array([[-1, -2, -INF, np.nan, -1], [-1, -1, -3, -2, -INF]], np.float32)
    got, val = select(vs, x, sc, 40)
    es, et, ep, _ = D.beam_select(val, sc, np.zeros((2, 5)), -1, 40)
    check(got, val, sc, 40)
    assert (got[1] == -1).any() and (got[0][got[1] == -1] == -INF).all() and (got[2][got[1] == -1] == -1).all()


def test_lowest_values_are_no_mask(vs):
    """The type's lowest finite value is a logit like any other."""
    x = np.full((2, 70), np.finfo(np.float32).min)
    x[1, 3] = 0
    sc = np.zeros((1, 2), np.float32)
    got, _ = select(vs, x, sc, 4)
    assert got[2].tolist() == [[1, 0, 0, 0]] and got[1].tolist() == [[3, 0, 1, 2]]


def test_finished_beams(vs):
    rng = np.random.default_rng(4)
    x, sc = rng.standard_normal((12, 901)), -20 * rng.random((3, 4)).astype(np.float32)
    fin = np.array([[0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0]], np.uint8)
    sc[0, 1] = -0.5
    x[8, 5] = 30  # a beam that ends now
    for eos in (5, 900, 901, -1):
        got, val = select(vs, x, sc, 6, finished=fin, eos=eos)
        check(got, val, sc, 6, fin, eos)
        if eos in (5, 900):
            assert got[1][0, 0] == eos and got[2][0, 0] == 1 and got[3][0, 0] == 1
            assert (got[1][1] >= 0).sum() == 4
        else:
            assert (got[1][1] == -1).all()


def test_refusals(vs):
    A = vs.DeviceArray
    bs = vs.BeamSearch()
    x, sc = A((6, 50), "f32"), A((2, 3), "f32")
    so, to, po = A((2, 4), "f32"), A((2, 4), "i32"), A((2, 4), "i32")
    for args in ((A((5, 50), "f32"), sc, so, to, po), (x, sc, so, A((2, 3), "i32"), po), (x, sc, so, A((2, 4), "f32"), po),
                 (A((6, 50), "i32"), sc, so, to, po), (View(x, (6, 50), (20, 1), 0), sc, so, to, po)):
        with pytest.raises(ValueError):
            bs.select(*args)
    with pytest.raises(NotImplementedError):
        bs.select(x, sc, A((2, 65), "f32"), A((2, 65), "i32"), A((2, 65), "i32"))
    with pytest.raises(NotImplementedError):
        bs.select(A((129, 5), "f32"), A((1, 129), "f32"), A((1, 2), "f32"), A((1, 2), "i32"), A((1, 2), "i32"))
    h = A((6, 8), "i32")
    for args in ((A((4,), "i32"), h, A((6, 8), "i32")), (A((6,), "i32"), h, A((6, 9), "i32")), (A((6,), "i32"), h, h),
                 (A((6,), "f32"), h, A((6, 8), "i32"))):
        with pytest.raises(ValueError):
            bs.reorder(*args)
    with pytest.raises(ValueError):
        bs.reorder(A((6,), "i32"), A((6, 8), "f32"), A((6, 8), "f32"), tail=A((6,), "i32"))
    bs.close()


def test_first_step(vs):
    """All beams equal, only the first alive."""
    rng = np.random.default_rng(6)
    row = rng.standard_normal(4000)
    sc = np.array([[0, -INF, -INF]], np.float32)
    got, val = select(vs, np.tile(row, (3, 1)), sc, 3)
    check(got, val, sc, 3)
    assert not got[2].any()


def test_large_logits(vs):
    """Values whose exponentials pass 32 bits."""
    rng = np.random.default_rng(8)
    x, sc = 1e4 * rng.standard_normal((4, 2500)), np.zeros((2, 2), np.float32)
    got, val = select(vs, x, sc, 4)
    es, et, ep, _ = D.beam_select(val, sc, np.zeros((2, 2)), -1, 4)
    assert np.array_equal(got[1], et) and np.array_equal(got[2], ep)
    # (the totals' rounding, and that of logits of this size)
    np.testing.assert_allclose(got[0], es, rtol=2.0 ** -22, atol=2.0 ** -18)


@pytest.mark.parametrize("dtype,npdt", [("i32", np.int32), ("f32", np.float32), ("bf16", np.uint16), ("u8", np.uint8)])
@pytest.mark.parametrize("cols", [1, 3, 16, 1024, 5000])
def test_reorder(vs, dtype, npdt, cols):
    rng = np.random.default_rng(cols)
    A = vs.DeviceArray
    state = rng.integers(0, 200, (7, cols)).astype(npdt)
    parents = np.array([6, 6, -1, 0, 7, 3, -2**31, 2], np.int32)
    out = A.of(np.full((8, cols), 9), dtype)
    bs = vs.BeamSearch()
    bs.reorder(A.of(parents, "i32"), A.of(state, dtype), out)
    ok = (parents >= 0) & (parents < 7)
    want = np.where(ok[:, None], state[np.where(ok, parents, 0)], 0)
    assert np.array_equal(out.numpy(), want)
    if dtype == "i32":
        tail = rng.integers(0, 99, 8)
        bs.reorder(A.of(parents.reshape(2, 4), "i32"), A.of(state, dtype), out, tail=A.of(tail.reshape(2, 4), "i32"))
        want[:, -1] = tail
        assert np.array_equal(out.numpy(), want)
    bs.close()
