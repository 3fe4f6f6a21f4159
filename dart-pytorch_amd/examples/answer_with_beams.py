"""Retrieve passages, then let a model answer with them: the index, the paged
cache, its attention and beam search as one program uses them.

The model is a stand-in with random weights whose projections run in numpy on
the host (a real one runs them on the GPU and hands the same buffers over);
search, cache, attention, the choice of the beams and the reordering of their
states run on the GPU.

  python dart-pytorch_amd/examples/answer_with_beams.py
"""
import os
import sys

import numpy as np

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

PAGE = 32


class Reader:
    """A small decoder: per layer attention with grouped heads and a tanh block."""

    def __init__(self, vocab=211, dim=64, layers=2, heads=4, kv_heads=2, head_dim=16, seed=0):
        g = np.random.default_rng(seed)
        w = lambda *s: (g.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)  # noqa: E731
        self.vocab, self.dim, self.layers = vocab, dim, layers
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.embed = g.standard_normal((vocab, dim)).astype(np.float32)
        self.place = g.standard_normal((4096, dim)).astype(np.float32) * 0.3
        self.wqkv = [w(dim, (heads + 2 * kv_heads) * head_dim) * 2 for _ in range(layers)]
        self.wo = [w(heads * head_dim, dim) for _ in range(layers)]
        self.w1 = [w(dim, dim) for _ in range(layers)]
        self.head = w(dim, vocab) * 3

    def enter(self, tokens, positions):
        return self.embed[tokens] + self.place[positions]

    def qkv(self, layer, x):
        """[rows, heads + 2 kv_heads, head_dim]: queries, keys and values side by side."""
        return (self.norm(x) @ self.wqkv[layer]).reshape(len(x), -1, self.head_dim)

    def leave(self, layer, x, attended):
        x = x + attended.reshape(len(x), -1) @ self.wo[layer]
        return x + np.tanh(self.norm(x) @ self.w1[layer])

    def logits(self, x):
        return self.norm(x) @ self.head

    @staticmethod
    def norm(x):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float32(1e-6))


def prompt_pass(model, tokens):
    """The prompt through the model on the host: each layer's keys and values, and the last position's logits."""
    x, rows, H, G = model.enter(tokens, np.arange(len(tokens))), [], model.heads, model.heads // model.kv_heads
    hidden = np.triu(np.ones((len(tokens),) * 2, bool), 1)
    for layer in range(model.layers):
        qkv = model.qkv(layer, x)
        q, k, v = qkv[:, :H], qkv[:, H:H + model.kv_heads], qkv[:, H + model.kv_heads:]
        s = np.einsum("qhd,khd->hqk", q, k.repeat(G, 1)) / np.sqrt(np.float32(model.head_dim))
        s = np.where(hidden, -np.inf, s)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        rows.append((k, v))
        x = model.leave(layer, x, np.einsum("hqk,khd->qhd", p, v.repeat(G, 1)).astype(np.float32))
    return rows, model.logits(x[-1:])


def answer(vs, model, prompt, beams=4, steps=12, eos=1, device=0):
    """The beams' tokens and scores after `steps` steps, best first."""
    A = vs.DeviceArray
    H, K, D = model.heads, model.kv_heads, model.head_dim
    width = -(-(len(prompt) + steps) // PAGE)
    pages = width + beams * (-(-steps // PAGE) + 2)
    cache = vs.PagedKVCache(pages, PAGE, K, D, layers=model.layers, dtype="f32", device=device)
    search = vs.BeamSearch(device)

    # the prompt: one sequence, its keys and values stored in bulk, shared by all beams
    rows, logits = prompt_pass(model, prompt)
    one = cache.new_sequences(1, width)
    cache.extend(one, len(prompt))
    for layer, (k, v) in enumerate(rows):
        cache.append(one, A.of(k, "f32"), A.of(v, "f32"), starts=A.of([0, len(prompt)], "i32"), layer=layer)
    seqs, spare = cache.new_sequences(beams, width, one.refs), cache.new_sequences(beams, width, one.refs)
    cache.fork(one, A.of(np.zeros(beams, np.int32), "i32"), seqs)

    scores = A.of(np.where(np.arange(beams) == 0, 0, -np.inf)[None], "f32")  # at first all beams are one
    ended = A.of(np.zeros((1, beams), np.uint8), "u8")
    next_scores, next_ended = A((1, beams), "f32"), A((1, beams), "u8")
    tokens, parents = A((1, beams), "i32"), A((1, beams), "i32")
    history = [A.of(np.full((beams, steps), eos, np.int32), "i32") for _ in range(2)]
    q, out = A((beams, H, D), "f32"), A((beams, H, D), "f32")
    k, v = A((beams, K, D), "f32"), A((beams, K, D), "f32")
    lg = A((beams, model.vocab), "f32").upload(np.tile(logits, (beams, 1)))
    for step in range(steps):
        search.select(lg, scores, next_scores, tokens, parents, finished=ended, finished_out=next_ended, eos=eos)
        # histories follow their parents and grow by a column
        search.reorder(parents, Columns(history[0], step + 1), Columns(history[1], step + 1), tail=tokens)
        history.reverse()
        cache.fork(seqs, parents, spare)
        seqs, spare = spare, seqs
        scores, next_scores, ended, next_ended = next_scores, scores, next_ended, ended
        if step + 1 == steps:
            break
        cache.extend(seqs, 1)
        x = model.enter(tokens.numpy()[0].clip(0), np.full(beams, len(prompt) + step))
        for layer in range(model.layers):
            qkv = model.qkv(layer, x)
            q.upload(qkv[:, :H]), k.upload(qkv[:, H:H + K]), v.upload(qkv[:, H + K:])
            cache.attend(seqs, q, out, k=k, v=v, layer=layer)
            x = model.leave(layer, x, out.numpy())
        lg.upload(model.logits(x))
        if step % 8 == 7:
            cache.compact(seqs)
    cache.check()
    result = history[0].numpy(), scores.numpy()[0]
    search.close()
    cache.close()
    return result


class Columns:
    """The first columns of a two-dimensional DeviceArray."""

    def __init__(self, base, n):
        self.base, self.shape, self.dtype = base, (base.shape[0], n), base.dtype

    def data_ptr(self):
        return self.base.data_ptr()

    def stride(self):
        return self.base.stride()


def retrieve(vs, question, embeddings, passages, k=2):
    """The tokens of the k passages nearest to the question."""
    index = vs.GpuIndexFlat.ip(embeddings.shape[1])
    index.add(embeddings)
    found = index.search(question[None], k).ids[0]
    index.close()
    return np.concatenate([passages[i] for i in found])


def main():
    import vector_store as vs

    g = np.random.default_rng(7)
    model = Reader()
    passages = [g.integers(2, model.vocab, n) for n in g.integers(10, 40, 50)]
    embeddings = g.standard_normal((50, 32)).astype(np.float32)
    question = embeddings[17] + 0.1 * g.standard_normal(32).astype(np.float32)
    prompt = np.concatenate([retrieve(vs, question, embeddings, passages), g.integers(2, model.vocab, 7)])
    tokens, scores = answer(vs, model, prompt)
    for row, score in zip(tokens, scores):
        print(f"{score:9.4f}  {' '.join(str(t) for t in row)}")


if __name__ == "__main__":
    main()
