"""A prompt's way through the operators together, as a program uses them: rows' places, rotated queries and keys
entering the cache, attention in chunks beside requests that decode, cross attention to passages' states, log
probabilities; against the same model on the host in 64 bits without a cache."""
import os
import sys

import numpy as np
import pytest

import _prompt as P

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dart-pytorch_amd", "examples"))


class Model:
    """The example's reader with rotary positions in place of learned ones, and a layer that attends to passages."""

    def __init__(self, ex, seed, dtype):
        self.r = ex.Reader(vocab=211, heads=4, kv_heads=2, head_dim=32, seed=seed)
        for name in ("embed", "head"):
            setattr(self.r, name, getattr(self.r, name).astype(dtype))
        for name in ("wqkv", "wo", "w1"):
            setattr(self.r, name, [w.astype(dtype) for w in getattr(self.r, name)])

    def qkv(self, layer, x):
        y = self.r.qkv(layer, x)
        return y[:, :4], y[:, 4:6], y[:, 6:]


def plain(m, tokens, states, w):
    """Logits of every position of one text; states: keys and values of its passages."""
    x, n = m.r.embed[tokens], len(tokens)
    for layer in range(2):
        q, k, v = m.qkv(layer, x)
        q, k = (P.turned(y, np.arange(n), w, 1.0, "half")[0] for y in (q, k))
        a = P.attend_rows(q, k, v, P.seen_mask(np.arange(n), n, 0, 0), 32 ** -0.5, "f32")[0]
        if layer == 0:
            a = a + P.attend_rows(q, states[0], states[1], np.ones((n, len(states[0])), bool), 32 ** -0.5, "f32")[0]
        x = m.r.leave(layer, x, a)
    return m.r.logits(x)


@pytest.mark.parametrize("seed", [0, 1])
def test_prompts_in_chunks_beside_decoding(vs, seed):
    import answer_with_beams as ex

    A, rng = vs.DeviceArray, np.random.default_rng(seed)
    m, exact = Model(ex, seed, np.float32), Model(ex, seed, np.float64)
    texts = [rng.integers(2, 211, n) for n in (150, 3, 70, 41)]
    # what each call brings of every text: chunks of prompts beside single tokens, and nothing at all
    plan = [[64, 1, 0, 17], [80, 1, 33, 1], [1, 0, 33, 1], [5, 1, 4, 22]]
    assert [sum(c) for c in zip(*plan)] == [len(t) for t in texts]
    rot = vs.Rotary(32, scaling="linear", factor=2.0)
    cache, beams = vs.PagedKVCache(40, 32, 2, 32, layers=2, dtype="f32"), vs.BeamSearch()
    seqs = cache.new_sequences(4, 6)
    # the passages' states: another set of sequences on the same pages
    lengths = [33, 5, 64, 90]
    states = [[rng.standard_normal((n, 2, 32)).astype(np.float32) for _ in range(2)] for n in lengths]
    passages = cache.new_sequences(4, 4, seqs.refs)
    cache.extend(passages, A.of(lengths, "i32"))
    starts = A((5,), "i32")
    cache.rows(passages, A.of(lengths, "i32"), starts)
    cache.append(passages, *(A.of(np.concatenate([s[i] for s in states]), "f32") for i in range(2)), starts=starts)
    done, got = [0] * 4, [[] for _ in texts]
    for counts in plan:
        rows = sum(counts)
        padded = rows + 3  # a batch may be filled up
        count = A.of(counts, "i32")
        cache.extend(seqs, count)
        sequence, position = A((padded,), "i32"), A((padded,), "i32")
        cache.rows(seqs, count, starts, sequence=sequence, position=position)
        b, p = sequence.numpy()[:rows], position.numpy()
        assert (p[rows:] == -1).all() and [list(b).count(i) for i in range(4)] == counts
        tokens = np.array([texts[i][j] for i, j in zip(b, p)])
        x = m.r.embed[np.concatenate([tokens, np.zeros(3, int)])]
        for layer in range(2):
            q, k, v = (A.of(y, "f32") for y in m.qkv(layer, x))
            out, cross = A.of(np.zeros((padded, 4, 32)), "f32"), A.of(np.zeros((padded, 4, 32)), "f32")
            cache.append(seqs, k, v, starts=starts, layer=layer, rotary=rot, q=q, q_out=q)
            cache.attend_rows(seqs, q, out, starts=starts, layer=layer)
            a = out.numpy()
            if layer == 0:
                cache.attend_rows(passages, q, cross, starts=starts, causal=False)
                a = a + cross.numpy()
            x = m.r.leave(layer, x, a)
        logits = m.r.logits(x).astype(np.float32)
        # each position's next token, where the text goes on
        nxt = np.array([texts[i][j + 1] if j + 1 < len(texts[i]) else -1 for i, j in zip(b, p)] + [-1] * 3)
        lp, ent = A((padded,), "f32"), A((padded,), "f32")
        top, tl = A((padded, 3), "i32"), A((padded, 3), "f32")
        beams.logprobs(A.of(logits, "f32"), A.of(nxt, "i32"), lp, entropy=ent, top_tokens=top, top_logprobs=tl)
        for i, j, row in zip(b, p, zip(lp.numpy(), ent.numpy(), top.numpy(), tl.numpy())):
            got[i].append(row)
            assert len(got[i]) == j + 1
    cache.check()
    for i, text in enumerate(texts):
        want = plain(exact, text, [s.astype(np.float64) for s in states[i]], rot.frequencies)
        lp, ent, tt, tl = P.logprobs(want, list(text[1:]) + [-1], 3)
        # 32-bit projections of two layers: 1e-5 of a logit of a few units, a few times over
        tol = 2e-5 * 8
        np.testing.assert_allclose([r[0] for r in got[i]], lp, rtol=0, atol=tol)
        np.testing.assert_allclose([r[1] for r in got[i]], ent, rtol=0, atol=tol * np.log(211))
        np.testing.assert_allclose([r[3] for r in got[i]], tl, rtol=0, atol=tol)
        near = np.diff(-tl, axis=1).min(1) > 2 * tol  # (tokens whose logits all but tie may change places)
        assert np.array_equal(np.array([r[2] for r in got[i]])[near, :2], tt[near, :2])
    cache.free(seqs)
    cache.free(passages)
    assert not seqs.refs.numpy().any()
