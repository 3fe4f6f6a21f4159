"""Plain forms of the decoding operators, in 64 bits with numpy: what the GPU
tests compare with.  Nothing here calls the library."""
import numpy as np


def to_bf16(x):
    """float -> bf16 bit patterns (uint16), nearest even; NaN stays NaN."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def stored(x, dtype):
    """x as the device holds it: (bits or floats to upload, the float32 values they stand for)"""
    if dtype == "bf16":
        b = to_bf16(x)
        return b, from_bf16(b)
    x = np.ascontiguousarray(x, np.float32)
    return x, x


def key_place(t, x, dim, dtype):
    e = 8 if dtype == "bf16" else 4
    return ((t // 16 * (dim // e) + x // e) * 16 + t % 16) * e + x % e


def value_place(t, x, dim, dtype):
    h, g, i = t // 16, t % 16 // 4, t % 4
    return ((x * 4 + g) * 2 + h) * 4 + i if dtype == "bf16" else ((h * dim + x) * 4 + g) * 4 + i


def places(dim, dtype):
    """[32, dim] places of a block's keys and values."""
    t, x = np.arange(32)[:, None], np.arange(dim)[None, :]
    return key_place(t, x, dim, dtype), value_place(t, x, dim, dtype)


def write_rows(pool, table, b, first, k, v, page, dtype):
    """Rows k, v [n, heads, dim] into pool [pages][2][heads][page * dim] at positions first.. of sequence b."""
    n, heads, dim = k.shape
    kp, vp = places(dim, dtype)
    for j in range(n):
        pos = first + j
        pg = table[b, pos // page]
        base, t = pos % page // 32 * 32 * dim, pos % 32
        pool[pg, 0][:, base + kp[t]] = k[j]
        pool[pg, 1][:, base + vp[t]] = v[j]


def visible(n, window, sinks):
    p = np.arange(n)
    return p if not window else p[(p >= n - window) | (p < sinks)]


def attend(q, k, v, seen, scale):
    """q [heads, dim], k, v [n, kv_heads, dim] float64; seen: positions.  (out, lse, bound of |scores|)"""
    heads, dim = q.shape
    kv = k.shape[1]
    out, lse = np.zeros((heads, dim)), np.full(heads, -np.inf)
    if len(seen) == 0:
        return out, lse
    for h in range(heads):
        g = h // (heads // kv)
        s = scale * (k[seen, g] @ q[h])
        m = s.max()
        p = np.exp(s - m)
        out[h] = (p / p.sum()) @ v[seen, g]
        lse[h] = m + np.log(p.sum())
    return out, lse


def attend_tolerance(q, k, v, seen, scale, dtype):
    """How far a correct result may be from attend()'s before its last rounding: (of out, of lse),
    both absolute.

    Scores: dim products summed in 32 bits by units that may truncate, off by at most
    (dim + 4) 2^-23 of the sum of the products' sizes, then the multiplications by scale * log2(e)
    (2^-22 of the score) and exp2 (2^-22).  A weight is off by that share and the sums over n
    positions and up to 400 partial sums by (n + 400) 2^-23 of the sum of the weights; bf16 weights
    are held to 2^-16.  The output is a weighted mean of values: twice the weights' error of the
    largest value."""
    if len(seen) == 0:
        return 0.0, 0.0
    dim = q.shape[1]
    size = np.abs(scale) * max(np.abs(k[seen, g]).dot(np.abs(q).max(0)).max() for g in range(k.shape[1]))
    ds = (dim + 4) * 2.0 ** -23 * size + 2.0 ** -21 * (size + 1)
    dw = ds + (len(seen) + 400) * 2.0 ** -23 + (2.0 ** -16 if dtype == "bf16" else 0)
    return np.abs(v[seen]).max() * 2 * dw, dw + 2.0 ** -21 * (size + 20)


def assert_rounded(got, exact, off, dtype, what=""):
    """Every value of `got` is what some number within `off` of `exact` rounds to in dtype."""
    low, high = stored(exact - off, dtype)[1], stored(exact + off, dtype)[1]
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), (what, got[bad][:5], exact[bad][:5], off)


# ------------------------------------------------------------------ pages


class Pages:
    """The page operators' rules, one sequence after the other."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs, self.page = (np.array(table), np.array(lens), np.array(refs), page)
        self.copies = []

    def extend(self, counts):
        n, width, page = len(self.lens), self.table.shape[1], self.page
        counts = np.maximum(np.broadcast_to(counts, n), 0)
        if any(c and ln + c > width * page for c, ln in zip(counts, self.lens)):
            return "width"
        last = [self.table[b, (ln - 1) // page] if c and ln % page else -1
                for b, (c, ln) in enumerate(zip(counts, self.lens))]
        shared = [b for b in range(n) if last[b] >= 0 and self.refs[last[b]] > 1]
        copy = set()
        for b in shared:
            holders = [x for x in shared if last[x] == last[b]]
            if holders[0] != b or len(holders) != self.refs[last[b]]:
                copy.add(b)
        want = [(b in copy) + -(-(ln + c) // page) - -(-ln // page) if c else 0
                for b, (c, ln) in enumerate(zip(counts, self.lens))]
        free = list(np.flatnonzero(self.refs == 0))
        if sum(want) > len(free):
            return "pages"
        for b in range(n):
            c, ln = int(counts[b]), int(self.lens[b])
            if not c:
                continue
            if b in copy:
                to = free.pop(0)
                self.copies.append((last[b], to))
                self.refs[last[b]] -= 1
                self.refs[to] = 1
                self.table[b, (ln - 1) // page] = to
            for e in range(-(-ln // page), -(-(ln + c) // page)):
                to = free.pop(0)
                self.refs[to] = 1
                self.table[b, e] = to
            self.lens[b] += c
        return None

    def fork(self, parents):
        table = np.full((len(parents), self.table.shape[1]), -1, np.int32)
        lens = np.zeros(len(parents), np.int32)
        refs = self.refs.copy()
        for row in self.table:
            np.subtract.at(refs, row[row >= 0], 1)
        for i, p in enumerate(parents):
            if p >= 0:
                table[i], lens[i] = self.table[p], self.lens[p]
                np.add.at(refs, table[i][table[i] >= 0], 1)
        return Pages(table, lens, refs, self.page)

    def compact(self):
        live = np.flatnonzero(self.refs)
        n = len(live)
        to = np.flatnonzero(self.refs[:n] == 0)
        src = live[live >= n]
        where = np.arange(len(self.refs))
        where[src] = to
        out = Pages(np.where(self.table >= 0, where[self.table], -1), self.lens, np.zeros_like(self.refs), self.page)
        out.refs[where[live]] = self.refs[live]
        out.copies = list(zip(src, to))
        return out


# ------------------------------------------------------------------- beams


def beam_select(logits, scores, finished, eos, k):
    """logits [requests * beams, vocab], scores and finished [requests, beams]; by the order
    (total, lower beam, larger logit, lower token).  Scores in 64 bits."""
    R, W = scores.shape
    V = logits.shape[1]
    out_s = np.full((R, k), -np.inf)
    out_t, out_p = np.full((R, k), -1, np.int64), np.full((R, k), -1, np.int64)
    out_f = np.zeros((R, k), np.uint8)
    for r in range(R):
        cand = []
        for w in range(W):
            sc = float(scores[r, w])
            x = logits[r * W + w].astype(np.float64)
            if np.isnan(sc) or sc == -np.inf:
                continue
            if finished[r, w]:
                if 0 <= eos < V:
                    cand.append((-sc, w, 0.0, eos))
                continue
            if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
                continue
            m = x.max()
            off = sc - np.log(np.exp(x - m).sum())  # (x - m first: x may be larger than scores by any amount)
            top = np.lexsort((np.arange(V), -x))[:k]
            cand += [(-(off + (x[t] - m)), w, -x[t], int(t)) for t in top if x[t] > -np.inf]
        for i, (s, w, _, t) in enumerate(sorted(cand)[:k]):
            out_s[r, i], out_t[r, i], out_p[r, i], out_f[r, i] = -s, t, r * W + w, t == eos
    return out_s, out_t, out_p, out_f
