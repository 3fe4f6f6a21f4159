"""The decoding calls on several streams at a time, each with work of its own, and recorded into graphs: every
result is that of the same call alone."""
import numpy as np
import pytest

import _decode as D
from _hip import Stream
from test_gpu_attend import Case

pytestmark = pytest.mark.gpu


def test_attention_on_streams_with_work_of_their_own(vs):
    """One handle; queries, lengths and numbers of sequences differ by stream, so do the partial sums in its scratch."""
    A = vs.DeviceArray
    lens = [4000, 9, 2500, 700, 3100, 64]
    c = Case(vs, lens, 8, 2, 64, 32, "bf16")
    plans = [[0, 1], [2, 3, 0, 4], [4], [5, 2, 0, 4, 3, 1], [3, 4]]
    work = []
    for i, plan in enumerate(plans):
        rows = np.array(plan)
        seqs = vs.KVSequences(A.of(c.table[rows], "i32"), A.of(c.lens[rows], "i32"), c.seqs.refs)
        qb, q = D.stored((1 + i) * c.rng.standard_normal((len(plan), 8, 64)), "bf16")
        outs = [(A((len(plan), 8, 64), "bf16"), A((len(plan), 8), "f32")) for _ in range(6)]
        work.append((plan, seqs, A.of(qb, "bf16"), q.astype(np.float64), outs, Stream()))
    for _, seqs, q, _, outs, st in work:  # (scratch exists, so that nothing waits below)
        c.cache.attend(seqs, q, outs[0][0], lse=outs[0][1], stream=st.ptr)
    for j in range(6):
        for _, seqs, q, _, outs, st in work:
            c.cache.attend(seqs, q, outs[j][0], lse=outs[j][1], stream=st.ptr)
    for w in work:
        w[5].sync()
    for plan, _, _, q, outs, _ in work:
        for out, lse in outs:
            o, el = D.from_bf16(out.numpy()), lse.numpy()
            for i, b in enumerate(plan):
                args = (q[i], c.k[b], c.v[b], np.arange(lens[b]), 64 ** -0.5)
                (eo, want), (to, tl) = D.attend(*args), D.attend_tolerance(*args, "bf16")
                D.assert_rounded(o[i], eo, to, "bf16", (plan, b))
                np.testing.assert_allclose(el[i], want, rtol=0, atol=tl)
            assert np.array_equal(out.numpy(), outs[0][0].numpy())


def test_pages_on_streams_with_work_of_their_own(vs):
    """One handle, sets of sequences with counts of their own: plans of extends, forks and compactions side by side."""
    A, npages, rng = vs.DeviceArray, 700, np.random.default_rng(4)
    cache = vs.PagedKVCache(npages, 32, 1, 16)
    work = []
    for i in range(4):
        n = 20 + 11 * i
        ids, lens = rng.permutation(npages // 4) + i * (npages // 4), rng.integers(1, 60, n)  # (pages apart: contents too)
        table = np.full((n, 5), -1, np.int32)
        at = 0
        for b in range(n):
            h = -(-int(lens[b]) // 32)
            table[b, :h] = ids[at:at + h]
            at += h
        refs = np.bincount(table[table >= 0], minlength=npages)
        refs[np.arange(npages) // (npages // 4) != i] += 1  # the other sets' pages are not to be had
        m = D.Pages(table, lens, refs, 32)
        put = lambda t, ln, r: vs.KVSequences(A.of(t, "i32"), A.of(ln, "i32"), A.of(r, "i32"))  # noqa: E731
        seqs, spare = put(table, lens, refs), put(np.full_like(table, 7), np.full(n, 7), np.full(npages, 7))
        parents = rng.integers(0, n, n)
        work.append((m, seqs, spare, parents, A.of(parents, "i32"), 1 + i, Stream()))
    for _, seqs, spare, _, parents, count, st in work:
        cache.fork(seqs, parents, spare, stream=st.ptr)
    for _ in range(3):
        for _, _, spare, _, _, count, st in work:
            cache.extend(spare, count, stream=st.ptr)
    for w in work:
        w[6].sync()
    for m, _, spare, parents, _, count, _ in work:
        m = m.fork(parents)
        for _ in range(3):
            assert m.extend(count) is None
        assert np.array_equal(spare.table.numpy(), m.table) and np.array_equal(spare.lens.numpy(), m.lens)
        assert np.array_equal(spare.refs.numpy(), m.refs)
    cache.check()


def test_selection_on_streams_with_work_of_their_own(vs):
    A, rng, bs = vs.DeviceArray, np.random.default_rng(5), vs.BeamSearch()
    work = []
    for i, (R, W, V, k) in enumerate([(1, 4, 50_001, 4), (3, 8, 9_000, 16), (2, 5, 30_000, 64), (4, 2, 2_100, 3)]):
        x, sc = 3 * rng.standard_normal((R * W, V)).astype(np.float32), -4 * rng.random((R, W)).astype(np.float32)
        outs = [(A((R, k), "f32"), A((R, k), "i32"), A((R, k), "i32")) for _ in range(5)]
        work.append((x, sc, k, A.of(x, "f32"), A.of(sc, "f32"), outs, Stream()))
    for j in (0, 0, 1, 2, 3, 4):
        for _, _, _, lg, sc, outs, st in work:
            bs.select(lg, sc, *outs[j], stream=st.ptr)
    for w in work:
        w[6].sync()
    for x, sc, k, _, _, outs, _ in work:
        es, et, ep, _ = D.beam_select(x, sc, np.zeros(sc.shape), -1, k)
        for so, to, po in outs:
            assert np.array_equal(to.numpy(), et) and np.array_equal(po.numpy(), ep)
            np.testing.assert_allclose(so.numpy(), es, rtol=2.0 ** -23, atol=2.0 ** -18)
    bs.close()


def test_selection_and_reordering_recorded_into_a_graph(vs):
    """Recorded once, replayed with other contents and eager calls between."""
    A, rng, bs, st = vs.DeviceArray, np.random.default_rng(6), vs.BeamSearch(), Stream()
    R, W, V, T = 3, 4, 20_011, 9
    lg, sc = A((R * W, V), "f32"), A((R, W), "f32")
    so, to, po = A((R, W), "f32"), A((R, W), "i32"), A((R, W), "i32")
    history, grown = A((R * W, T), "i32"), A((R * W, T), "i32")
    eager = A((R, W), "f32"), A((R, W), "i32"), A((R, W), "i32")

    def step():
        bs.select(lg, sc, so, to, po, stream=st.ptr)
        bs.reorder(po, history, grown, tail=to, stream=st.ptr)

    st.begin()
    try:
        with pytest.raises(NotImplementedError, match="scratch"):
            bs.select(lg, sc, so, to, po, stream=st.ptr)
        bs.reorder(po, history, grown, tail=to, stream=st.ptr)
    finally:
        st.end()
    lg.upload(np.zeros((R * W, V))), sc.upload(np.zeros((R, W)))
    step()
    st.sync()
    st.begin()
    step()
    graph = st.end()
    for i in range(5):
        x = 3 * rng.standard_normal((R * W, V)).astype(np.float32)
        scores, h = -4 * rng.random((R, W)).astype(np.float32), rng.integers(0, V, (R * W, T))
        lg.upload(x), sc.upload(scores), history.upload(h)
        st.replay(graph)
        es, et, ep, _ = D.beam_select(x, scores, np.zeros((R, W)), -1, W)
        assert np.array_equal(to.numpy(), et) and np.array_equal(po.numpy(), ep), i
        np.testing.assert_allclose(so.numpy(), es, rtol=2.0 ** -23, atol=2.0 ** -18)
        want = h[ep.ravel()]
        want[:, -1] = et.ravel()
        assert np.array_equal(grown.numpy(), want)
        bs.select(lg, sc, *eager)  # (the default stream's own scratch)
        assert np.array_equal(eager[0].numpy(), so.numpy()) and np.array_equal(eager[1].numpy(), et)
    bs.close()


def test_attention_and_compaction_recorded_with_the_new_token(vs):
    """A step that stores its token and a compaction, replayed."""
    c = Case(vs, [90, 31, 64], 4, 2, 64, 32, "bf16", width=300)
    refs = np.bincount(c.table[c.table >= 0], minlength=c.cache.npages).astype(np.int32)
    c.sequences(refs)
    A, st = vs.DeviceArray, Stream()
    q, out = A.of(c.qb, "bf16"), A((3, 4, 64), "bf16")
    k, v = A((3, 2, 64), "bf16"), A((3, 2, 64), "bf16")

    def step():
        c.cache.attend(c.seqs, q, out, k=k, v=v, stream=st.ptr)
        c.cache.compact(c.seqs, stream=st.ptr)

    k.upload(np.zeros((3, 2, 64))), v.upload(np.zeros((3, 2, 64)))
    step()
    st.sync()
    st.begin()
    step()
    graph = st.end()
    for i in range(4):
        c.qb, x = D.stored(c.rng.standard_normal((3, 4, 64)), "bf16")
        (kb, kx), (vb, vx) = (D.stored(c.rng.standard_normal((3, 2, 64)), "bf16") for _ in range(2))
        c.q = x.astype(np.float64)
        q.upload(c.qb), k.upload(kb), v.upload(vb)
        st.replay(graph)
        for b in range(3):
            c.k[b][-1], c.v[b][-1] = kx[b], vx[b]
        c.compare((D.from_bf16(out.numpy()), c.run()[1]))
    c.cache.check()


def test_same_bits_whatever_ran_before(vs):
    """What earlier calls leave in the scratch changes nothing."""
    c = Case(vs, [3000, 17, 900, 5000], 8, 2, 64, 32, "bf16")
    refs = np.bincount(c.table[c.table >= 0], minlength=c.cache.npages).astype(np.int32)
    c.sequences(refs)
    first = c.run()
    other = Case(vs, [5000, 5000], 8, 2, 64, 32, "bf16", seed=1)
    other.cache = c.cache  # (its own sequences on the same handle: whatever pages they name)
    A = vs.DeviceArray
    table = np.where(other.table < c.cache.npages, other.table, -1)
    other.seqs = vs.KVSequences(A.of(table, "i32"), A.of(other.lens, "i32"), c.seqs.refs)
    for _ in range(3):
        other.run()
        c.cache.compact(c.seqs, c.seqs)
        again = c.run()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
