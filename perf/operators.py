"""Performance cases of the decoding operators: attention of one new token over a
paged key-value cache, the cache's pages, and beam search's selection.

Each case is one step that a program takes while it generates text: attention
of every sequence's new token (which is stored in the same call), forking the
cache along the beams' parents and giving every sequence its next position,
compacting the cache, or choosing the next beams and reordering their
histories.  Sizes are generic.

  listed()           the named cases
  draw(rng)          one more case of the same ranges
  prepare(case, s)   inputs of seed s on the GPU
  run(state)         one pass: the plain form, or the library where `own` is set
  work(case)         bytes and operations one pass cannot do without
  exact(case, s)     the floating results in 64 bits

Pages.  A page holds the keys and values of `page` consecutive positions of one
sequence, for every layer and key-value head, in blocks of 32 positions.  With
E = 16 / element size, position t = 16 h + 4 g + i of a block (h < 2, g < 4,
i < 4) and dimension x:
  pool    [page id][layer][0: keys, 1: values][head][block][32 * dim]
  keys    [h][x // E][4 g + i][x % E]
  values  bf16: [x][g][h][i]     fp32: [h][x][g][i]
"""
import math
import os
import sys

import torch

DEV = "cuda:0"

own = False


def listed():
    return [
        # one user's chat, a thousand positions in: latency is all
        {"name": "attend_chat", "kind": "attend", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "min_len": 1000, "max_len": 1000, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a serving batch of requests of very different lengths
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "min_len": 65, "max_len": 8190, "window": 0, "sinks": 0, "dtype": "bf16"},
        # two long documents: few rows, the length has to be split
        {"name": "attend_long", "kind": "attend", "seqs": 2, "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 128, "min_len": 120_001, "max_len": 131_072, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a small model in fp32 with one key-value head per query head
        {"name": "attend_f32", "kind": "attend", "seqs": 16, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 64, "min_len": 17, "max_len": 1023, "window": 0, "sinks": 0, "dtype": "f32"},
        # sliding-window layers of long requests, the first positions always visible
        {"name": "attend_window", "kind": "attend", "seqs": 32, "heads": 24, "kv_heads": 4, "dim": 96,
         "page": 64, "min_len": 900, "max_len": 30_000, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # one request's four beams: the cache follows the beams' parents
        {"name": "fork_four", "kind": "fork", "requests": 1, "beams": 4, "layers": 12, "kv_heads": 12,
         "dim": 64, "page": 32, "prompt": 300, "new": 21, "pages": 96, "dtype": "bf16"},
        # 64 requests of four beams each over long shared prompts
        {"name": "fork_batch", "kind": "fork", "requests": 64, "beams": 4, "layers": 8, "kv_heads": 8,
         "dim": 128, "page": 32, "prompt": 1000, "new": 45, "pages": 3500, "dtype": "bf16"},
        # a small cache after a few requests have ended
        {"name": "compact_small", "kind": "compact", "seqs": 8, "layers": 12, "kv_heads": 12, "dim": 64,
         "page": 32, "shared": 4, "each": 9, "pages": 150, "dtype": "bf16"},
        # a server's cache, half empty: the live pages move to its front
        {"name": "compact_large", "kind": "compact", "seqs": 96, "layers": 8, "kv_heads": 8, "dim": 128,
         "page": 32, "shared": 10, "each": 21, "pages": 4100, "dtype": "bf16"},
        # one request, four beams, a vocabulary of odd size
        {"name": "beam_four", "kind": "beam", "requests": 1, "beams": 4, "vocab": 50_001, "k": 4,
         "time": 37, "dtype": "f32"},
        # a batch of five beams each, ten candidates: those that end leave five to go on with
        {"name": "beam_ten", "kind": "beam", "requests": 16, "beams": 5, "vocab": 32_000, "k": 10,
         "time": 250, "dtype": "bf16"},
        # large batch, many beams, large vocabulary
        {"name": "beam_batch", "kind": "beam", "requests": 64, "beams": 8, "vocab": 128_000, "k": 8,
         "time": 1023, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["fork"] * 2 + ["compact"] * 2 + ["beam"] * 3)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    size = 2 if dtype == "bf16" else 4
    if kind == "attend":
        kv, dim = rng.choice([1, 2, 4, 5, 8, 12, 16]), rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
        per_kv = rng.choice([1, 1, 2, 3, 4, 4, 6, 8, 8, 16])
        seqs = _log(rng, 1, 256)
        # at most a billion bytes of cache, were every sequence of the greatest length
        most = max(64, min(131_072, int(1e9 / (seqs * kv * dim * 2 * size))))
        high = _log(rng, 33, most)
        window = rng.choice([0, 0, 0, _log(rng, 1, 5000)])
        return {"kind": "attend", "seqs": seqs, "heads": kv * per_kv, "kv_heads": kv, "dim": dim,
                "page": rng.choice([32, 32, 64, 128]), "min_len": _log(rng, 1, high), "max_len": high,
                "window": window, "sinks": rng.choice([0, 1, 4, 40]) if window else 0, "dtype": dtype}
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 16])
        vocab = _log(rng, 500, 160_000)
        requests = max(1, min(_log(rng, 1, 128), int(6.5e7 / (beams * vocab))))
        return {"kind": "beam", "requests": requests, "beams": beams, "vocab": vocab,
                "k": rng.choice([beams, beams, 2 * beams]), "time": _log(rng, 1, 1023), "dtype": dtype}
    layers, kv, dim, page = rng.choice([1, 4, 8, 12, 24]), rng.choice([2, 4, 8, 12]), rng.choice([64, 80, 128]), rng.choice([32, 64])
    bytes_ = layers * 2 * kv * page * dim * size
    if kind == "fork":
        beams, prompt, new = rng.choice([2, 3, 4, 5, 8]), _log(rng, 1, 2000), _log(rng, 1, 200)
        each = prompt // page + beams * (-(-(prompt % page + new) // page) + 2)
        requests = max(1, min(_log(rng, 1, 80), int(3e9 / (each * bytes_))))
        return {"kind": "fork", "requests": requests, "beams": beams, "layers": layers, "kv_heads": kv, "dim": dim,
                "page": page, "prompt": prompt, "new": new, "pages": requests * each + rng.randrange(9), "dtype": dtype}
    seqs, shared, each = _log(rng, 1, 100), rng.randrange(12), _log(rng, 1, 40)
    seqs = max(1, min(seqs, int(1.3e9 / (each * bytes_))))
    live = shared + seqs * each
    return {"kind": "compact", "seqs": seqs, "layers": layers, "kv_heads": kv, "dim": dim, "page": page,
            "shared": shared, "each": each, "pages": int(live * rng.uniform(1.1, 2.5)) + 1, "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _lens(case):
    """Lengths between min_len and max_len, spread over their logarithm.  They go by the
    sequence's place alone, so that the work is the same for every seed."""
    at = torch.arange(case["seqs"], dtype=torch.float64)
    u = torch.frac(at * 0.6180339887498949 + 0.75)
    low, high = math.log(case["min_len"]), math.log(case["max_len"])
    return torch.exp(low + u * (high - low)).round().to(torch.int64)


def _visible(case):
    """How many positions each sequence's new token attends to."""
    n = _lens(case)
    if not case["window"]:
        return n
    seen = n.clamp(max=case["window"])
    return seen + (n - seen).clamp(max=case["sinks"])


def _pool(case, pages, layers, seed):
    shape = (pages, layers, 2, case["kv_heads"], case["page"] * case["dim"])
    return torch.randn(shape, device=DEV, dtype=_dtype(case), generator=_gen(seed, 1))


def _prepare_attend(case, seed):
    n, page = _lens(case), case["page"]
    held = -(-n // page)
    width, total = int(held.max()), int(held.sum())
    # pages were given out as the sequences grew, so theirs lie anywhere in the pool
    ids = torch.randperm(total + 3, device=DEV, generator=_gen(seed, 2))[:total].to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < held.to(DEV)[:, None]] = ids
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    # the projection's output row: queries, keys and values of one token side by side
    qkv = torch.randn(case["seqs"], H + 2 * Hk, D, device=DEV, generator=_gen(seed, 3))
    qkv[:, :H] *= 2.0
    qkv = qkv.to(_dtype(case))
    return {"pool": _pool(case, total + 3, 1, seed), "table": table, "lens": n.to(torch.int32).to(DEV),
            "refs": torch.zeros(total + 3, dtype=torch.int32, device=DEV).index_fill_(0, ids.long(), 1),
            "q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:],
            "out": torch.empty(case["seqs"], H, D, device=DEV, dtype=_dtype(case)),
            "lse": torch.empty(case["seqs"], H, device=DEV)}


def _prepare_fork(case, seed):
    R, W, page, P = case["requests"], case["beams"], case["page"], case["pages"]
    length = case["prompt"] + case["new"]
    common, held = case["prompt"] // page, -(-length // page)
    ids = torch.randperm(P, device=DEV, generator=_gen(seed, 2)).to(torch.int32)
    width = held + 3
    table = torch.full((R, W, width), -1, dtype=torch.int32, device=DEV)
    # the prompt's full pages are one for all beams of a request, the rest is each beam's own
    table[:, :, :common] = ids[:R * common].view(R, 1, common)
    table[:, :, common:held] = ids[R * common:R * (common + W * (held - common))].view(R, W, held - common)
    table = table.view(R * W, width)
    refs = torch.bincount(table[table >= 0].long(), minlength=P).to(torch.int32)
    # a quarter of the beams end here and as many go on twice; which ones, goes by the seed
    mixed = torch.rand(R, W, device=DEV, generator=_gen(seed, 4)).argsort(1)
    local = mixed[:, torch.arange(W, device=DEV) * 3 // 4]
    parents = (local + torch.arange(R, device=DEV)[:, None] * W).to(torch.int32).view(-1)
    return {"pool": _pool(case, P, case["layers"], seed), "table": table, "refs": refs, "parents": parents,
            "lens": torch.full((R * W,), length, dtype=torch.int32, device=DEV),
            "table2": torch.empty_like(table), "refs2": torch.empty_like(refs),
            "lens2": torch.empty(R * W, dtype=torch.int32, device=DEV)}


def _prepare_compact(case, seed):
    S, P, common, each = case["seqs"], case["pages"], case["shared"], case["each"]
    ids = torch.randperm(P, device=DEV, generator=_gen(seed, 2)).to(torch.int32)
    table = torch.full((S, common + each + 2), -1, dtype=torch.int32, device=DEV)
    table[:, :common] = ids[:common]
    table[:, common:common + each] = ids[common:common + S * each].view(S, each)
    refs = torch.bincount(table[table >= 0].long(), minlength=P).to(torch.int32)
    lens = torch.full((S,), (common + each) * case["page"] - 5, dtype=torch.int32, device=DEV)
    return {"pool": _pool(case, P, case["layers"], seed), "table": table, "refs": refs, "lens": lens,
            "table2": torch.empty_like(table), "refs2": torch.empty_like(refs), "lens2": torch.empty_like(lens)}


def _logits(case, seed):
    """Logits of a head: spread by 2.5, a few likely tokens well above the rest.  Beams are at scores
    between -30 and -2, and some have ended."""
    R, W, V, g = case["requests"], case["beams"], case["vocab"], _gen(seed, 3)
    x = torch.randn(R * W, V, device=DEV, generator=g).mul_(2.5)
    likely = torch.randint(0, V, (R * W, 5), device=DEV, generator=g)
    x.scatter_(1, likely, 8.0 + 4.0 * torch.rand(R * W, 5, device=DEV, generator=g))
    # on a grid of 1/1024: tokens of one beam tie exactly, or lie apart
    x = x.mul_(1024.0).round_().div_(1024.0).to(_dtype(case))
    ended = torch.rand(R, W, device=DEV, generator=g) < 0.1
    return x, ended


def _totals(x, scores, ended, eos):
    """Scores of all continuations, [requests, beams * vocab], in the type of `x`."""
    R, W = scores.shape
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    total = scores.reshape(-1, 1) + (x - lse)
    stay = torch.full_like(total, -math.inf)
    stay[:, eos] = scores.reshape(-1)
    return torch.where(ended.reshape(-1, 1), stay, total).view(R, -1)


def _prepare_beam(case, seed):
    R, W, V, k, T = case["requests"], case["beams"], case["vocab"], case["k"], case["time"]
    x, ended = _logits(case, seed)
    eos, g = 2, _gen(seed, 4)
    scores = -2.0 - 28.0 * torch.rand(R, W, device=DEV, generator=g)
    # Which of two beams' continuations is better is not told by 32 bits where their scores all
    # but tie: those requests' scores are drawn again.  Exact ties within a beam stay.
    for _ in range(20):
        best = _totals(x.double(), scores.double(), ended, eos).topk(min(k + 1, W * V), 1)
        near = (best.values[:, :-1] - best.values[:, 1:]).abs() < 1e-3
        near &= best.indices[:, :-1] // V != best.indices[:, 1:] // V
        again = -2.0 - 28.0 * torch.rand(R, W, device=DEV, generator=g)
        scores = torch.where(near.any(1, keepdim=True), again, scores)
        if not near.any():
            break
    history = torch.randint(0, V, (R * W, T + 1), device=DEV, generator=g, dtype=torch.int32)
    i32 = {"dtype": torch.int32, "device": DEV}
    return {"x": x, "scores": scores, "ended": ended.to(torch.uint8), "eos": eos, "history": history,
            "scores2": torch.empty(R, k, device=DEV), "tokens2": torch.empty(R, k, **i32),
            "parents2": torch.empty(R, k, **i32), "ended2": torch.empty(R, k, dtype=torch.uint8, device=DEV),
            "history2": torch.empty(R * k, T + 1, **i32)}


def prepare(case, seed):
    make = {"attend": _prepare_attend, "fork": _prepare_fork, "compact": _prepare_compact, "beam": _prepare_beam}
    s = make[case["kind"]](case, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------- plain form


def _keys(pool, case):
    """[page][layer][head][block][h][x // E][t % 16][x % E]"""
    e = 16 // pool.element_size()
    return pool[:, :, 0].view(pool.shape[0], pool.shape[1], case["kv_heads"], case["page"] // 32, 2, case["dim"] // e, 16, e)


def _values(pool, case):
    """[page][layer][head][block], then bf16 [x][g][h][i] or fp32 [h][x][g][i]"""
    inner = (case["dim"], 4, 2, 4) if pool.dtype == torch.bfloat16 else (2, case["dim"], 4, 4)
    return pool[:, :, 1].view(pool.shape[0], pool.shape[1], case["kv_heads"], case["page"] // 32, *inner)


def _rows_at(view, pool, case, page, pos, is_value):
    """Keys or values at positions `pos` of pages `page` (same shape): [..., heads, dim]"""
    block, t = pos % case["page"] // 32, pos % 32
    if is_value and pool.dtype == torch.bfloat16:
        return view[page, 0, :, block, :, t % 16 // 4, t // 16, t % 4]
    if is_value:
        return view[page, 0, :, block, t // 16, :, t % 16 // 4, t % 4]
    return view[page, 0, :, block, t // 16, :, t % 16, :].flatten(-2)


def _plain_attend(s):
    case, pool, table = s["case"], s["pool"], s["table"].long()
    B, Hk, D = case["seqs"], case["kv_heads"], case["dim"]
    n, W, S = s["lens"].long(), case["window"], case["sinks"]
    K, V = _keys(pool, case), _values(pool, case)
    # the new token's keys and values go to each sequence's last position
    last = n - 1
    page, block, t = table.gather(1, last[:, None] // case["page"])[:, 0], last % case["page"] // 32, last % 32
    K[page, 0, :, block, t // 16, :, t % 16, :] = s["k"].unflatten(-1, (-1, K.shape[-1]))
    if pool.dtype == torch.bfloat16:
        V[page, 0, :, block, :, t % 16 // 4, t // 16, t % 4] = s["v"]
    else:
        V[page, 0, :, block, t // 16, :, t % 16 // 4, t % 4] = s["v"]
    # the positions that some sequence sees, and which of them each does
    if W:
        pos = torch.cat([torch.arange(S, device=DEV).expand(B, S), n[:, None] - W + torch.arange(W, device=DEV)], 1)
        seen = (pos < n[:, None]) & (pos >= torch.where(torch.arange(S + W, device=DEV) < S, 0, S))
    else:
        pos = torch.arange(case["max_len"], device=DEV).expand(B, -1)
        seen = pos < n[:, None]
    pos = torch.where(seen, pos, 0)
    page = table.gather(1, pos // case["page"])
    k = _rows_at(K, pool, case, page, pos, False).float().transpose(1, 2).contiguous()  # [B, Hk, N, D]
    v = _rows_at(V, pool, case, page, pos, True).float().transpose(1, 2).contiguous()
    q = s["q"].float().view(B, Hk, -1, D).transpose(2, 3).contiguous()
    x = torch.matmul(k, q) / math.sqrt(D)  # [B, Hk, N, G]
    x = x.masked_fill(~seen[:, None, :, None], -math.inf)
    top = x.amax(2, keepdim=True)
    p = (x - top).exp()
    total = p.sum(2, keepdim=True)
    out = torch.matmul((p / total).transpose(2, 3).contiguous(), v)  # [B, Hk, G, D]
    return {"out": out.reshape(B, -1, D).to(_dtype(case)), "lse": (top + total.log()).reshape(B, -1), "pool": pool}


def _plain_fork(s):
    case, pool, P, page = s["case"], s["pool"], s["case"]["pages"], s["case"]["page"]
    parents = s["parents"].long()
    # every chosen sequence's entries gain a reference, every sequence given up takes its own away
    table, lens = s["table"][parents], s["lens"][parents].long()
    children = torch.bincount(parents, minlength=s["table"].shape[0]) - 1
    held = s["table"] >= 0
    gain = torch.where(held, children[:, None], 0).view(-1)
    refs = s["refs"].long().index_add_(0, s["table"].long().clamp(min=0).view(-1), gain)
    # one more position each: a new page where the last is full; a copy of it where others hold it too
    # (the first of its holders keeps it if they all go on)
    full, at = lens % page == 0, (lens - 1) // page
    last = table.gather(1, at[:, None]).long()[:, 0]
    shared = ~full & (refs[last] > 1)
    holders = torch.bincount(last[shared], minlength=P)
    order = torch.arange(len(lens), device=DEV)
    first = torch.full((P,), len(lens), device=DEV).scatter_reduce_(0, last, torch.where(shared, order, len(lens)), "amin")
    copy = shared & ~((first[last] == order) & (holders[last] == refs[last]))
    need = full | copy
    free = (refs != 0).to(torch.int8).argsort(stable=True)
    new = free[(need.cumsum(0) - 1).clamp(min=0)]
    pool[new[copy]] = pool[last[copy]]
    refs.index_add_(0, last, -copy.long()).index_add_(0, new, need.long())
    at = torch.where(full, lens // page, at)
    table = table.scatter(1, at[:, None], torch.where(need, new, last).to(torch.int32)[:, None])
    return {"table": table, "lens": (lens + 1).to(torch.int32), "refs": refs.to(torch.int32), "pool": pool}


def _plain_compact(s):
    pool, refs, table = s["pool"], s["refs"], s["table"]
    live = refs > 0
    front = torch.arange(len(refs), device=DEV) < live.sum()
    to, start = (front & ~live).nonzero()[:, 0], (~front & live).nonzero()[:, 0]
    pool[to] = pool[start]
    moved = torch.arange(len(refs), device=DEV, dtype=torch.int32)
    moved[start] = to.to(torch.int32)
    refs2 = torch.where(front, refs, 0)
    refs2[to] = refs[start]
    return {"table": torch.where(table >= 0, moved[table.clamp(min=0).long()], -1), "lens": s["lens"], "refs": refs2, "pool": pool}


def _plain_beam(s):
    case, W, V = s["case"], s["case"]["beams"], s["case"]["vocab"]
    total = _totals(s["x"].float(), s["scores"], s["ended"] != 0, s["eos"])
    # the k best, ties to the lowest place: score and place make one whole number
    bits = total.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    place = torch.arange(W * V, device=DEV)
    at = (bits * 2**31 + (2**31 - 1 - place)).topk(case["k"], 1).indices
    scores = total.gather(1, at)
    none = scores == -math.inf
    beam = at // V
    parents = (beam + torch.arange(len(at), device=DEV)[:, None] * W).masked_fill(none, -1)
    tokens = (at % V).masked_fill(none, -1)
    ended = (tokens == s["eos"]) & ~none
    rows = s["history"][parents.clamp(min=0).view(-1)]
    rows = torch.where(none.view(-1, 1), 0, rows)
    rows[:, -1] = tokens.view(-1)
    return {"scores": scores, "tokens": tokens.to(torch.int32), "parents": parents.to(torch.int32),
            "ended": ended.to(torch.uint8), "history": rows.to(torch.int32)}


# -------------------------------------------------------- the library's calls


def _cache(s):
    """The cache over the state's pool and the sequences on it, as a program keeps them."""
    if "cache" not in s:
        root = os.path.join(os.getcwd(), "dart-pytorch_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        import vector_store as vs

        s["vs"], case = vs, s["case"]
        if "pool" in s:
            pool = s["pool"]
            s["cache"] = vs.PagedKVCache(pool.shape[0], case["page"], case["kv_heads"], case["dim"], layers=pool.shape[1],
                                         dtype=case["dtype"], memory=pool)
            s["seqs"] = vs.KVSequences(s["table"], s["lens"], s["refs"])
            if "table2" in s:
                s["seqs2"] = vs.KVSequences(s["table2"], s["lens2"], s["refs2"])
        else:
            s["cache"] = vs.BeamSearch()
    return s["cache"]


def _own_attend(s):
    case = s["case"]
    _cache(s).attend(s["seqs"], s["q"], s["out"], k=s["k"], v=s["v"], lse=s["lse"], window=case["window"],
                     sinks=case["sinks"], stream=torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"], "lse": s["lse"], "pool": s["pool"]}


def _own_fork(s):
    cache, stream = _cache(s), torch.cuda.current_stream().cuda_stream
    cache.fork(s["seqs"], s["parents"], s["seqs2"], stream=stream)
    cache.extend(s["seqs2"], 1, stream=stream)
    return {"table": s["table2"], "lens": s["lens2"], "refs": s["refs2"], "pool": s["pool"]}


def _own_compact(s):
    _cache(s).compact(s["seqs"], s["seqs2"], stream=torch.cuda.current_stream().cuda_stream)
    return {"table": s["table2"], "lens": s["lens2"], "refs": s["refs2"], "pool": s["pool"]}


def _own_beam(s):
    beams, stream = _cache(s), torch.cuda.current_stream().cuda_stream
    beams.select(s["x"], s["scores"], s["scores2"], s["tokens2"], s["parents2"], finished=s["ended"],
                 finished_out=s["ended2"], eos=s["eos"], stream=stream)
    beams.reorder(s["parents2"], s["history"], s["history2"], tail=s["tokens2"], stream=stream)
    return {"scores": s["scores2"], "tokens": s["tokens2"], "parents": s["parents2"], "ended": s["ended2"],
            "history": s["history2"]}


def run(s):
    if own:
        return {"attend": _own_attend, "fork": _own_fork, "compact": _own_compact, "beam": _own_beam}[s["case"]["kind"]](s)
    return {"attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact, "beam": _plain_beam}[s["case"]["kind"]](s)


# ------------------------------------------------------------- accounting


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "attend":
        seen, D = int(_visible(case).sum()), case["dim"]
        rows = case["seqs"] * (2 * case["heads"] + 4 * case["kv_heads"]) * D * size  # q, out; new k and v read and stored
        return {"bytes": seen * case["kv_heads"] * 2 * D * size + rows + case["seqs"] * case["heads"] * 4,
                "flops": 4.0 * seen * case["heads"] * D}
    if case["kind"] == "beam":
        R, W, k = case["requests"], case["beams"], case["k"]
        return {"bytes": R * W * case["vocab"] * size + R * (W * 5 + k * 13) + R * k * (case["time"] + 1) * 8,
                "flops": 4.0 * R * W * case["vocab"]}
    page = case["layers"] * 2 * case["kv_heads"] * case["page"] * case["dim"] * size
    if case["kind"] == "fork":
        rows = case["requests"] * case["beams"]
        length = case["prompt"] + case["new"]
        # in each request, beams * 3 // 4 of the old sequences (rounded up) go on, the others are copies
        kept = (case["beams"] - 1) * 3 // 4 + 1
        copies = case["requests"] * (case["beams"] - kept) if length % case["page"] else 0
        width = -(-length // case["page"]) + 3
        return {"bytes": copies * 2 * page + (rows * (width + 1) + case["pages"]) * 8 + rows * 4, "flops": 0}
    live = case["shared"] + case["seqs"] * case["each"]
    moves = live * (1.0 - live / case["pages"])  # of pages that lie anywhere, on average
    return {"bytes": moves * 2 * page + (case["seqs"] * (case["shared"] + case["each"] + 3) + case["pages"]) * 8, "flops": 0}


# ---------------------------------------------------------- 64-bit results


def _exact_attend(case, seed):
    s = prepare(case, seed)
    Hk, D, page = case["kv_heads"], case["dim"], case["page"]
    E = 16 // s["pool"].element_size()
    outs, lses = [], []
    for b, n in enumerate(_lens(case).tolist()):
        ids = s["table"][b, :-(-n // page)].long()
        raw = s["pool"][ids, 0].double()  # [pages, 2, Hk, page * D]
        k = raw[:, 0].reshape(-1, Hk, page // 32, 2, D // E, 16, E).permute(1, 0, 2, 3, 5, 4, 6).reshape(Hk, -1, D)
        if case["dtype"] == "bf16":
            v = raw[:, 1].reshape(-1, Hk, page // 32, D, 4, 2, 4).permute(1, 0, 2, 5, 4, 6, 3).reshape(Hk, -1, D)
        else:
            v = raw[:, 1].reshape(-1, Hk, page // 32, 2, D, 16).permute(1, 0, 2, 3, 5, 4).reshape(Hk, -1, D)
        k, v = k[:, :n].clone(), v[:, :n].clone()
        k[:, -1], v[:, -1] = s["k"][b].double(), s["v"][b].double()
        at = torch.arange(n, device=DEV)
        if case["window"]:
            at = at[(at >= n - case["window"]) | (at < case["sinks"])]
        k, v = k[:, at], v[:, at]
        q = s["q"][b].double().view(Hk, -1, D)
        x = torch.bmm(q, k.transpose(1, 2).contiguous()) * D ** -0.5
        lse = torch.logsumexp(x, 2, keepdim=True)
        outs.append(torch.bmm((x - lse).exp(), v).view(-1, D))
        lses.append(lse.view(-1))
    return {"out": torch.stack(outs), "lse": torch.stack(lses), "pool": None}


def _exact_beam(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    logp = x - torch.logsumexp(x, 1, keepdim=True) + s["scores"].double().view(-1, 1)
    over = torch.full_like(logp, -math.inf)
    over[:, s["eos"]] = s["scores"].double().view(-1)
    logp = torch.where((s["ended"] != 0).view(-1, 1), over, logp).view(case["requests"], -1)
    best = logp.sort(1, descending=True).values[:, :case["k"]] if logp.numel() < 1 << 20 else logp.topk(case["k"], 1).values
    return {"scores": best, "tokens": None, "parents": None, "ended": None, "history": None}


def exact(case, seed):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "beam":
        return _exact_beam(case, seed)
    return None  # pages and whole numbers: nothing is rounded
