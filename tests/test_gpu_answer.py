"""Retrieval, cache, attention and beam search together, as the example runs them, against the same search
without a cache: every beam's whole text through the model on the host, in 64 bits."""
import os
import sys

import numpy as np
import pytest

import _decode as D

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dart-pytorch_amd", "examples"))


def plain(ex, model, prompt, beams, steps, eos):
    for name in ("embed", "place", "head"):
        setattr(model, name, getattr(model, name).astype(np.float64))
    for name in ("wqkv", "wo", "w1"):
        setattr(model, name, [w.astype(np.float64) for w in getattr(model, name)])
    texts, scores, ended = [[] for _ in range(beams)], np.full((1, beams), -np.inf), np.zeros((1, beams), np.uint8)
    scores[0, 0] = 0
    for _ in range(steps):
        logits = np.concatenate([ex.prompt_pass(model, np.concatenate([prompt, np.array(t, int)]))[1] for t in texts])
        scores, tokens, parents, ended = D.beam_select(logits, scores, ended, eos, beams)
        texts = [texts[p] + [int(t)] for p, t in zip(parents[0], tokens[0])]
    return np.array(texts), scores[0]


@pytest.mark.parametrize("seed,length,beams,steps,eos", [(0, 61, 4, 20, 1), (1, 31, 3, 12, 5), (2, 96, 5, 9, 2), (3, 1, 2, 40, 1)])
def test_example_equals_the_search_without_a_cache(vs, seed, length, beams, steps, eos):
    import answer_with_beams as ex

    prompt = np.random.default_rng(seed).integers(2, 211, length)
    tokens, scores = ex.answer(vs, ex.Reader(seed=seed), prompt, beams, steps, eos)
    want, ws = plain(ex, ex.Reader(seed=seed), prompt, beams, steps, eos)
    assert np.array_equal(tokens, want)
    # 32-bit projections of two layers: 1e-5 of a logit of a few units, summed over the steps
    np.testing.assert_allclose(scores, ws, rtol=0, atol=2e-5 * steps * 8)


def test_retrieval_feeds_the_prompt(vs, capsys):
    import answer_with_beams as ex

    ex.main()
    out = capsys.readouterr().out.split("\n")
    assert len([line for line in out if line.strip()]) == 4
