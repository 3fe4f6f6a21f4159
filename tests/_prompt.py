"""Plain forms of the operators that a prompt passes through, in 64 bits with
numpy: what the GPU tests compare with.  Nothing here calls the library."""
import math

import numpy as np


def seen_mask(last, n, window, sinks):
    """[rows, n]: whether the row whose last position is last[i] sees position p (window 0: all up to it)."""
    p, t = np.arange(n)[None, :], np.asarray(last)[:, None]
    seen = p <= t
    return seen & ((p > t - window) | (p < sinks)) if window else seen


def attend_rows(q, k, v, seen, scale, dtype):
    """q [rows, heads, dim], k, v [n, kv_heads, dim] float64, seen [rows, n].

    (out, lse, how far a correct result may be from out before its last rounding, and from lse)

    Scores: dim products summed in 32 bits by units that may truncate, off by at most (dim + 4) 2^-23 of the sum of
    the products' sizes; scale * log2(e) and its product with them 2^-22 of the score, exp2 2^-22.  A weight is off by
    that share, the sums over n positions and their parts by (n + 400) 2^-23 of the sum of the weights.  The output is
    a weighted mean of values: twice the weights' error of the largest value.  bf16: each weight is rounded to bf16
    besides, half a step, 2^-8 of it, and divided by the sum of what they are rounded to: with p (1 + d) for p and out =
    sum of p v, the output moves by sum of p d (v - out) over 1 + sum of p d, at most 2^-8 (1 + 2^-7) of the sum of
    p (|v| + |out|)."""
    rows, heads, dim = q.shape
    kv, n = k.shape[1], k.shape[0]
    out, lse = np.zeros((rows, heads, dim)), np.full((rows, heads), -np.inf)
    off, loff = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    for h in range(heads):
        g = h // (heads // kv)
        hit = seen.any(0)
        s = scale * (q[:, h] @ k[hit, g].T)
        s = np.where(seen[:, hit], s, -np.inf)
        some = seen.any(1)
        if not some.any():
            continue
        m = np.where(some, s.max(1, initial=-np.inf), 0)[:, None]
        p = np.exp(s - m)
        total = p.sum(1, keepdims=True)
        p = p / np.where(total > 0, total, 1)
        out[:, h] = p @ v[hit, g]
        lse[some, h] = (m + np.log(np.where(total > 0, total, 1)))[some, 0]
        size = np.abs(scale) * np.abs(k[hit, g]).dot(np.abs(q[:, h]).T).max(0)
        ds = (dim + 4) * 2.0 ** -23 * size + 2.0 ** -21 * (size + 1)
        dw = ds + (n + 400) * 2.0 ** -23
        off[:, h] = (np.abs(v[hit, g]).max() * 2 * dw)[:, None]
        if dtype == "bf16":
            off[:, h] += 2.0 ** -8 * (1 + 2.0 ** -7) * (1 + dw[:, None]) * (p @ np.abs(v[hit, g]) + np.abs(out[:, h]))
        loff[:, h] = dw + 2.0 ** -21 * (size + 20)
    return out, lse, off, loff


def turned(x, positions, w, gain, layout, backward=False):
    """x [rows, heads, dim] float64 turned by positions times w (radians per position); the size that rounding
    errors of its values go by comes second."""
    dims = 2 * len(w)
    y, size = x.copy(), np.abs(x)
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if layout == "half" else (slice(0, dims, 2), slice(1, dims, 2))
    # (the angle's whole turns are taken off in whole numbers: 64 bits lose nothing of far positions)
    angle = np.array([[math.fmod(int(p) * wi, 2 * math.pi) for wi in w] for p in positions]).reshape(-1, 1, len(w))
    c, s = gain * np.cos(angle), gain * np.sin(angle) * (-1 if backward else 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = abs(gain) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


def turn_tolerance(size, positions, w):
    """Before the last rounding.  Cosine and sine: the angle's 2^-32 turns that are cut off (1.5e-9 radians), its own
    rounding and the polynomials' (below 4 roundings of values up to 1, and what they leave out, 1.8e-9), the gain's
    product: 6 2^-24 + 4e-9 in all; two products and a sum 3 2^-24.  The reference's angle is a 64-bit product: 2^-52 of
    it, and so is the frequency in turns."""
    far = np.abs(np.asarray(positions, np.float64)).max(initial=0) * np.abs(w).max(initial=0)
    return (9 * 2.0 ** -24 + 4e-9 + far * 2.0 ** -51) * size


def rows_of(counts, lens, table, page, npages, nrows):
    """(starts, sequence, position, slot) of vs_kv_rows, one row after the other."""
    counts = np.maximum(np.asarray(counts, np.int64), 0)
    starts = np.concatenate([[0], counts.cumsum()])
    out = np.full((3, nrows), -1, np.int64)
    for b in range(len(counts)):
        for i in range(starts[b], min(starts[b + 1], nrows)):
            out[0, i] = b
            pos = int(lens[b]) - (starts[b + 1] - i)
            if pos < 0:
                continue
            out[1, i] = pos
            if pos // page < table.shape[1] and 0 <= table[b, pos // page] < npages:
                out[2, i] = int(table[b, pos // page]) * page + pos % page
    return (np.minimum(starts, 2**31 - 1),) + tuple(out)


def logprobs(x, tokens, k):
    """(log probabilities, entropy, top tokens, their log probabilities) of rows of float64 logits."""
    rows, vocab = x.shape
    lp, ent = np.full(rows, np.nan), np.full(rows, np.nan)
    tt, tl = np.full((rows, k), -1, np.int64), np.full((rows, k), -np.inf)
    for i in range(rows):
        t = int(tokens[i])
        if t == -1:
            lp[i] = 0
        m = x[i].max()
        if np.isnan(x[i]).any() or np.isinf(m):
            continue
        e = np.exp(x[i] - m)
        log_s = np.log(e.sum())
        ent[i] = log_s - (e[e > 0] * (x[i] - m)[e > 0]).sum() / e.sum()
        if 0 <= t < vocab:
            lp[i] = (x[i, t] - m) - log_s
        best = np.lexsort((np.arange(vocab), -x[i]))[:k]
        best = best[x[i, best] > -np.inf]
        tt[i, :len(best)], tl[i, :len(best)] = best, (x[i, best] - m) - log_s
    return lp, ent, tt, tl
