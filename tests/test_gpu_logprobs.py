"""Log probabilities of given tokens, entropies and alternatives against their
definition in 64 bits."""
import numpy as np
import pytest

import _decode as D
import _prompt as P
from _hip import Stream
from test_gpu_attend import View

pytestmark = pytest.mark.gpu


def run(vs, bs, xb, dtype, tokens, k, logits=None, stream=0):
    A, rows = vs.DeviceArray, len(tokens)
    lp, ent = A.of(np.full(rows, 7.0), "f32"), A.of(np.full(rows, 7.0), "f32")
    tt, tl = A.of(np.full((rows, k), 7), "i32"), A.of(np.full((rows, k), 7.0), "f32")
    bs.logprobs(A.of(xb, dtype) if logits is None else logits, A.of(tokens, "i32"), lp, entropy=ent,
                top_tokens=tt if k else None, top_logprobs=tl if k else None, stream=stream)
    return [x.numpy() for x in (lp, ent, tt, tl)]


def compare(got, x, tokens, k):
    """Sums of v exponentials in 32 bits, a lane's share one after the other (v / 64 of them and 64 more steps of
    joining at most): each off by 2^-24 of the sum; exp2 by 2^-22 of its value, its argument by 2^-23 of the
    exponent, of which what counts is below 104 (smaller exponentials are 0).  log s is off by that share; the
    entropy's sum of e d by as much of sum of e |d| and 2^-23 more, that is of the entropy and log s together."""
    rows, vocab = x.shape
    lp, ent, tt, tl = P.logprobs(x.astype(np.float64), tokens, k)
    share = (vocab / 64 + 80) * 2.0 ** -24 + 2.0 ** -22
    with np.errstate(all="ignore"):
        d = x.astype(np.float64) - x.max(1, keepdims=True)
        e = np.exp(d)
        p = e / e.sum(1, keepdims=True)
        bend = np.nan_to_num((p * np.abs(np.where(p > 0, d, 0)) * 2.0 ** -22).sum(1))  # the arguments' roundings
        far = np.nan_to_num((p * np.where(p > 0, d, 0) ** 2 * 2.0 ** -22).sum(1))
    off = share + bend
    for have, want, more in ((got[0], lp, 0), (got[1], ent, off * (np.abs(np.nan_to_num(ent)) + np.log(vocab) + 1) + far)):
        assert np.array_equal(np.isnan(have), np.isnan(want)) and np.array_equal(np.isinf(have), np.isinf(want))
        fine = np.isfinite(want)
        err = np.abs(have[fine] - want[fine])
        assert (err <= (off + more)[fine] + np.abs(want[fine]) * 2.0 ** -24).all(), err.max()
    assert np.array_equal(got[2], tt)
    fine = np.isfinite(tl)
    assert np.array_equal(fine, np.isfinite(got[3])) and (got[3][~fine] == -np.inf).all()
    err = np.abs(got[3] - np.where(fine, tl, got[3]))
    assert (np.nan_to_num(err) <= off[:, None] + np.abs(np.where(fine, tl, 0)) * 2.0 ** -24).all()


VOCABS = [1, 2, 7, 63, 64, 65, 511, 512, 1023, 1024, 1025, 4095, 4096, 4097, 8193, 50001]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_vocabularies(vs, dtype, vocab):
    bs, rng = vs.BeamSearch(), np.random.default_rng(vocab)
    for rows, k in ((1, 0), (3, 5), (17, 1), (2, 64)):
        xb, x = D.stored(rng.standard_normal((rows, vocab)) * 3, dtype)
        tokens = rng.integers(-1, vocab, rows)
        compare(run(vs, bs, xb, dtype, tokens, k), x, tokens, k)
    bs.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("k", [0, 3, 40])
def test_large_calls(vs, dtype, k):
    """Long steps; rows enough for a workgroup each, and fewer."""
    bs, rng = vs.BeamSearch(), np.random.default_rng(k)
    for rows, vocab in ((600, 30011), (9000, 2000)):
        xb, x = D.stored(rng.standard_normal((rows, vocab), np.float32) * 2, dtype)
        tokens = rng.integers(0, vocab, rows)
        compare(run(vs, bs, xb, dtype, tokens, k), x, tokens, k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ties_go_to_the_lowest_token(vs, dtype):
    bs = vs.BeamSearch()
    for vocab, levels in ((3000, 1), (20000, 3), (9000, 40)):
        rng = np.random.default_rng(vocab)
        xb, x = D.stored(rng.integers(0, levels, (5, vocab)) * 0.25, dtype)
        for k in (1, 17, 64):
            compare(run(vs, bs, xb, dtype, np.arange(5), k), x, np.arange(5), k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5000])
def test_masks_and_rows_without_a_distribution(vs, dtype, vocab):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, vocab)).astype(np.float32) * 4
    x[0, rng.permutation(vocab)[: vocab - 3]] = -np.inf   # three left
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, vocab // 2] = 3                                   # certain
    x[3, vocab - 1] = np.nan
    x[4, 0] = np.inf
    x[5] = np.finfo(np.float32).min if dtype == "f32" else -3.3895314e38
    x[6, :vocab // 2] = -np.inf
    x[7] = 1e4 + x[7]                                      # large logits cost no digits
    x[8] = 0
    xb, x = D.stored(x, dtype)
    tokens = np.array([1, 0, vocab // 2, 3, 5, 7, 0, vocab - 1, 9])
    compare(run(vs, vs.BeamSearch(), xb, dtype, tokens, 7), x, tokens, 7)


def test_tokens_out_of_range(vs):
    xb, x = D.stored(np.random.default_rng(6).standard_normal((6, 100)), "f32")
    tokens = np.array([-1, -2, 100, 99, 2**31 - 1, -2**31])
    got = run(vs, vs.BeamSearch(), xb, "f32", tokens, 0)
    assert got[0][0] == 0 and np.isnan(got[0][[1, 2, 4, 5]]).all()
    compare(got, x, tokens, 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strided_rows_any_alignment(vs, dtype):
    A, rng = vs.DeviceArray, np.random.default_rng(7)
    rows, vocab, wide = 5, 3001, 3010
    xb, x = D.stored(rng.standard_normal((rows, wide)), dtype)
    base, tokens = A.of(xb, dtype), rng.integers(0, vocab, rows)
    for offset in (0, 1, 9):
        view = View(base, (rows, vocab), (wide, 1), offset)
        got = run(vs, vs.BeamSearch(), None, dtype, tokens, 4, logits=view)
        compare(got, x[:, offset:offset + vocab], tokens, 4)


def test_the_same_as_beam_search(vs):
    """A request of one beam at score 0: its k best totals are the k best log probabilities, to the bit."""
    A, rng, bs = vs.DeviceArray, np.random.default_rng(8), vs.BeamSearch()
    xb, x = D.stored(rng.standard_normal((6, 5000)) * 3, "bf16")
    got = run(vs, bs, xb, "bf16", np.zeros(6, int), 5)
    s, t, p = A((6, 5), "f32"), A((6, 5), "i32"), A((6, 5), "i32")
    bs.select(A.of(xb, "bf16"), A.of(np.zeros((6, 1)), "f32"), s, t, p)
    assert np.array_equal(t.numpy(), got[2])
    np.testing.assert_allclose(s.numpy(), got[3], rtol=0, atol=2 * (5000 / 64 + 80) * 2.0 ** -24 + 2.0 ** -20)


def test_streams_and_graphs(vs):
    A, rng, bs = vs.DeviceArray, np.random.default_rng(9), vs.BeamSearch()
    xb, x = D.stored(rng.standard_normal((30, 9000)) * 3, "bf16")
    tokens = rng.integers(0, 9000, 30)
    want, st = run(vs, bs, xb, "bf16", tokens, 4), Stream()
    logits, tok = A.of(xb, "bf16"), A.of(tokens, "i32")
    outs = [A((30,), "f32"), A((30,), "f32"), A((30, 4), "i32"), A((30, 4), "f32")]
    call = lambda: bs.logprobs(logits, tok, outs[0], entropy=outs[1], top_tokens=outs[2], top_logprobs=outs[3], stream=st.ptr)  # noqa: E731
    st.begin()
    with pytest.raises(NotImplementedError, match="scratch"):
        call()
    st.end()
    call()
    st.sync()
    st.begin()
    call()
    graph = st.end()
    for _ in range(3):
        for o in outs:
            o.upload(np.zeros(o.shape))
        run(vs, bs, xb, "bf16", tokens[::-1].copy(), 4)
        st.replay(graph)
        assert all(np.array_equal(o.numpy(), w) for o, w in zip(outs, want))


def test_refusals(vs):
    A, bs = vs.DeviceArray, vs.BeamSearch()
    x, tok, out = A((4, 100), "f32"), A.of(np.zeros(4), "i32"), A((4,), "f32")
    tt, tl = A((4, 3), "i32"), A((4, 3), "f32")
    for args, kw in (((x, tok, None), {}), ((x, None, out), {}), ((x, A((3,), "i32"), out), {}), ((x, tok, A((4,), "i32")), {}),
                     ((x, tok, out), dict(entropy=out)), ((x, tok, out), dict(top_tokens=tt)),
                     ((x, tok, out), dict(top_tokens=tt, top_logprobs=A((4, 2), "f32"))),
                     ((A((4, 100), "i32"), tok, out), {}), ((x, tok, View(x, (4,), (1,), 0)), {}),
                     ((x, tok, out), dict(entropy=A((4, 1), "f32")))):
        with pytest.raises(ValueError):
            bs.logprobs(*args, **kw)
    with pytest.raises(NotImplementedError):
        bs.logprobs(x, tok, out, top_tokens=A((4, 65), "i32"), top_logprobs=A((4, 65), "f32"))
    bs.logprobs(x, None, None, entropy=out, top_tokens=tt, top_logprobs=tl)
    bs.logprobs(A((0, 100), "f32"), A((0,), "i32"), A((0,), "f32"))
