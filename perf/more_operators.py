"""Performance cases of what a prompt passes through before the first decoding step:
where its tokens go in the paged key-value cache, their rotary positions, attention of
many new tokens at once, and the log probabilities that a model gives to them.

Each case is one step that a program takes with a batch of requests, some of which
bring one new token and some thousands: the rows' places from the requests' counts,
rotating queries and keys and storing keys and values, attention of all rows over the
cache, or scoring given tokens by their logits.  Sizes are generic.

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
        # a long prompt as one chunk, nothing before it: products are all
        {"name": "attend_prompt", "kind": "attend", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "min_len": 8192, "max_len": 8192, "min_rows": 8192, "max_rows": 8192, "every": 1, "causal": True,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # a serving batch: every 16th request brings a chunk of its prompt, the others decode
        {"name": "attend_mixed", "kind": "attend", "seqs": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "min_len": 600, "max_len": 8190, "min_rows": 1, "max_rows": 511, "every": 16, "causal": True,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # a few drafted tokens of each of a few long requests, to be accepted or not
        {"name": "attend_drafts", "kind": "attend", "seqs": 4, "heads": 32, "kv_heads": 4, "dim": 128, "page": 32,
         "min_len": 900, "max_len": 30_000, "min_rows": 5, "max_rows": 5, "every": 1, "causal": True,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # sliding-window layers, chunks of prompts that are far along, the first positions always visible
        {"name": "attend_window", "kind": "attend", "seqs": 4, "heads": 24, "kv_heads": 4, "dim": 96, "page": 64,
         "min_len": 3000, "max_len": 20_000, "min_rows": 700, "max_rows": 1500, "every": 1, "causal": True,
         "window": 2048, "sinks": 4, "dtype": "bf16"},
        # whole short prompts of a small model in fp32, one key-value head per query head
        {"name": "attend_f32", "kind": "attend", "seqs": 6, "heads": 12, "kv_heads": 12, "dim": 64, "page": 32,
         "min_len": 17, "max_len": 1023, "min_rows": 1023, "max_rows": 1023, "every": 1, "causal": True,
         "window": 0, "sinks": 0, "dtype": "f32"},
        # cross attention: the rows of an answer over the states of retrieved passages
        {"name": "attend_passages", "kind": "attend", "seqs": 16, "heads": 16, "kv_heads": 16, "dim": 64, "page": 32,
         "min_len": 200, "max_len": 4000, "min_rows": 40, "max_rows": 130, "every": 1, "causal": False,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # one decoding step's new tokens: rotated and stored, a part of the head, interleaved pairs
        {"name": "enter_step", "kind": "enter", "seqs": 48, "heads": 12, "kv_heads": 12, "dim": 64, "page": 32,
         "min_len": 20, "max_len": 1000, "min_rows": 1, "max_rows": 1, "part": 32, "layout": "interleaved",
         "scaling": "none", "factor": 1.0, "original": 0, "dtype": "f32"},
        # chunks of prompts far along a context that is longer than the model's own
        {"name": "enter_prompts", "kind": "enter", "seqs": 6, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "min_len": 5000, "max_len": 60_000, "min_rows": 500, "max_rows": 4100, "part": 128, "layout": "half",
         "scaling": "ramp", "factor": 8.0, "original": 8192, "dtype": "bf16"},
        # where the rows of a small batch go
        {"name": "rows_batch", "kind": "rows", "seqs": 48, "min_len": 65, "max_len": 8190, "min_rows": 1,
         "max_rows": 300, "every": 8, "page": 32, "spare": 70},
        # where the rows of very many requests go
        {"name": "rows_many", "kind": "rows", "seqs": 3000, "min_len": 30, "max_len": 4000, "min_rows": 1,
         "max_rows": 512, "every": 12, "page": 64, "spare": 1000},
        # the tokens of a few drafts with their alternatives, a vocabulary of odd size
        {"name": "score_drafts", "kind": "score", "rows": 20, "vocab": 50_001, "k": 5, "dtype": "f32"},
        # a passage scored token by token
        {"name": "score_passage", "kind": "score", "rows": 2048, "vocab": 128_000, "k": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["enter"] * 2 + ["rows"] + ["score"] * 2)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    size = 2 if dtype == "bf16" else 4
    if kind == "score":
        vocab = _log(rng, 500, 160_000)
        rows = max(1, min(_log(rng, 1, 4096), int(4e8 / (vocab * size))))
        return {"kind": "score", "rows": rows, "vocab": vocab, "k": rng.choice([0, 0, 1, 5, 20]), "dtype": dtype}
    if kind == "rows":
        high = _log(rng, 1, 2000)
        return {"kind": "rows", "seqs": _log(rng, 1, 8000), "min_len": high, "max_len": 2 * high, "min_rows": 1,
                "max_rows": _log(rng, 1, min(high, 256)), "every": rng.choice([1, 2, 8, 30]),
                "page": rng.choice([32, 64, 128]), "spare": _log(rng, 1, 500)}
    kv, dim = rng.choice([1, 2, 4, 5, 8, 12, 16]), rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([32, 32, 64, 128])
    if kind == "enter":
        heads, high = kv * rng.choice([1, 1, 2, 3, 4, 8]), _log(rng, 33, 60_000)
        rows = _log(rng, 1, min(high, 4000))
        seqs = max(1, min(_log(rng, 1, 100), int(1.5e8 / (rows * (heads + kv) * dim * size)),
                          int(8e8 / (high * kv * dim * 2 * size))))
        part = rng.choice([dim, dim, dim // 2, dim // 4])
        scaling = rng.choice(["none", "none", "linear", "base", "ramp"])
        return {"kind": "enter", "seqs": seqs, "heads": heads, "kv_heads": kv, "dim": dim, "page": page,
                "min_len": rng.randint(max(1, high // 3), high), "max_len": high, "min_rows": rng.randint(1, rows),
                "max_rows": rows, "part": part, "layout": rng.choice(["half", "interleaved"]), "scaling": scaling,
                "factor": rng.choice([2.0, 4.0, 8.0, 32.0]) if scaling != "none" else 1.0,
                "original": rng.choice([2048, 8192]) if scaling == "ramp" else 0, "dtype": dtype}
    heads = kv * rng.choice([1, 1, 2, 3, 4, 4, 6, 8, 8, 16])
    seqs = _log(rng, 1, 48)
    # at most a billion bytes of cache, were every sequence of the greatest length
    high = _log(rng, 33, max(64, min(60_000, int(1e9 / (seqs * kv * dim * 2 * size)))))
    causal = rng.choice([True, True, True, False])
    window = _log(rng, 1, 4000) if causal and rng.random() < 0.3 else 0
    # a quarter of the largest listed case's products
    most = max(1.0, 2.5e11 / (8 if dtype == "f32" else 1) / (4.0 * high * heads * dim))
    rows = _log(rng, 1, max(1, min(high, int(most), 4000)))
    every = rng.choice([1, 1, 1, 4, 16])
    seqs = max(1, min(seqs, int(most / rows * every)))
    return {"kind": "attend", "seqs": seqs, "heads": heads, "kv_heads": kv, "dim": dim, "page": page,
            "min_len": rng.randint(max(1, high // 10), high), "max_len": high,
            "min_rows": 1 if every > 1 else rng.randint(1, rows), "max_rows": rows, "every": every, "causal": causal,
            "window": window, "sinks": rng.choice([0, 1, 4, 40]) if window else 0, "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _spread(n, low, high, shift):
    """n whole numbers between low and high, spread over their logarithm.  They go by their place
    alone, so that the work is the same for every seed."""
    u = torch.frac(torch.arange(n, dtype=torch.float64) * 0.6180339887498949 + shift)
    return torch.exp(math.log(low) + u * (math.log(high) - math.log(low))).round().to(torch.int64)


def _sizes(case):
    """Each sequence's length, and how many of its last positions are new."""
    n = _spread(case["seqs"], case["min_len"], case["max_len"], 0.75)
    every = case.get("every", 1)
    if every > 1:  # every so many sequences bring a chunk, the others one row
        c = torch.full_like(n, case["min_rows"])
        c[every // 2::every] = case["max_rows"]
    else:
        c = _spread(case["seqs"], case["min_rows"], case["max_rows"], 0.3)
    return n, torch.minimum(c, n)


def _starts(c):
    return torch.cat([torch.zeros(1, dtype=torch.int64), c.cumsum(0)])


def _table(case, n, seed):
    """Pages were given out as the sequences grew, so theirs lie anywhere in the pool."""
    held = -(-n // case["page"])
    width, total = int(held.max()), int(held.sum())
    ids = torch.randperm(total + 3, device=DEV, generator=_gen(seed, 2))[:total].to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < held.to(DEV)[:, None]] = ids
    refs = torch.zeros(total + 3, dtype=torch.int32, device=DEV).index_fill_(0, ids.long(), 1)
    return table, refs


def _on_cache(case, seed):
    """Sequences on a cache of one layer, and the rows of a projection: queries, keys and values side by side."""
    n, c = _sizes(case)
    table, refs = _table(case, n, seed)
    H, Hk, D, R = case["heads"], case["kv_heads"], case["dim"], int(c.sum())
    qkv = torch.randn(R, H + 2 * Hk, D, device=DEV, generator=_gen(seed, 3))
    qkv[:, :H] *= 2.0
    qkv = qkv.to(_dtype(case))
    pool = torch.randn((refs.shape[0], 1, 2, Hk, case["page"] * D), device=DEV, dtype=_dtype(case), generator=_gen(seed, 1))
    return {"pool": pool, "table": table, "lens": n.to(torch.int32).to(DEV), "refs": refs,
            "starts": _starts(c).to(torch.int32).to(DEV), "sizes": (n.tolist(), c.tolist(), _starts(c).tolist()),
            "q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:],
            "out": torch.empty(R, H, D, device=DEV, dtype=_dtype(case))}


def _prepare_attend(case, seed):
    s = _on_cache(case, seed)
    s["lse"] = torch.empty(s["out"].shape[:2], device=DEV)
    return s


def _prepare_rows(case, seed):
    n, c = _sizes(case)
    # which sequence has which length and brings how many goes by the seed
    mixed = torch.randperm(case["seqs"], device=DEV, generator=_gen(seed, 4)).cpu()
    n, c = n[mixed], c[mixed]
    table, refs = _table(case, n, seed)
    rows = int(c.sum()) + case["spare"]  # a batch is filled up to a size of its own
    i32 = {"dtype": torch.int32, "device": DEV}
    return {"table": table, "lens": n.to(torch.int32).to(DEV), "refs": refs, "counts": c.to(torch.int32).to(DEV),
            "starts": torch.empty(case["seqs"] + 1, **i32), "sequence": torch.empty(rows, **i32),
            "position": torch.empty(rows, **i32), "slot": torch.empty(rows, **i32)}


def _prepare_score(case, seed):
    """Logits of a head: spread by 2.5, a few likely tokens well above the rest; most given tokens are
    likely ones, some rows have none."""
    R, V, g = case["rows"], case["vocab"], _gen(seed, 5)
    x = torch.randn(R, V, device=DEV, generator=g).mul_(2.5)
    likely = torch.randint(0, V, (R, 5), device=DEV, generator=g)
    x.scatter_(1, likely, 8.0 + 4.0 * torch.rand(R, 5, device=DEV, generator=g))
    x = x.to(_dtype(case))
    token = torch.where(torch.rand(R, device=DEV, generator=g) < 0.7, likely[:, 0],
                        torch.randint(0, V, (R,), device=DEV, generator=g))
    token = torch.where(torch.arange(R, device=DEV) % 32 == 31, -1, token).to(torch.int32)
    k = case["k"]
    return {"x": x, "token": token, "logprob": torch.empty(R, device=DEV), "entropy": torch.empty(R, device=DEV),
            "top": torch.empty(R, k, dtype=torch.int32, device=DEV), "top_logprob": torch.empty(R, k, device=DEV)}


def prepare(case, seed):
    make = {"attend": _prepare_attend, "enter": _on_cache, "rows": _prepare_rows, "score": _prepare_score}
    s = make[case["kind"]](case, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------- plain form


def _held(pool, case, pages, n):
    """Keys and values [kv_heads, n, dim] of a sequence on these pages, in 32 bits."""
    Hk, D, blocks = case["kv_heads"], case["dim"], case["page"] // 32
    e = 16 // pool.element_size()
    raw = pool[pages, 0]
    k = raw[:, 0].view(-1, Hk, blocks, 2, D // e, 16, e).permute(1, 0, 2, 3, 5, 4, 6).reshape(Hk, -1, D)
    if pool.dtype == torch.bfloat16:
        v = raw[:, 1].view(-1, Hk, blocks, D, 4, 2, 4).permute(1, 0, 2, 5, 4, 6, 3).reshape(Hk, -1, D)
    else:
        v = raw[:, 1].view(-1, Hk, blocks, 2, D, 16).permute(1, 0, 2, 3, 5, 4).reshape(Hk, -1, D)
    return k[:, :n].float(), v[:, :n].float()


def _plain_attend(s):
    case, out, lse = s["case"], s["out"], s["lse"]
    Hk, D, W = case["kv_heads"], case["dim"], case["window"]
    G = case["heads"] // Hk
    for b, (n, c, at) in enumerate(zip(*s["sizes"])):
        k, v = _held(s["pool"], case, s["table"][b, :-(-n // case["page"])].long(), n)
        q = s["q"][at:at + c].float().view(c, Hk, G, D).transpose(0, 1).reshape(Hk, c * G, D)
        x = torch.matmul(q, k.transpose(1, 2)).div_(math.sqrt(D)).view(Hk, c, G, n)
        if case["causal"]:
            row, pos = torch.arange(n - c, n, device=DEV)[:, None], torch.arange(n, device=DEV)
            hidden = pos > row
            if W:
                hidden |= (pos <= row - W) & (pos >= case["sinks"])
            x.masked_fill_(hidden[:, None, :], -math.inf)
        top = x.amax(3, keepdim=True)
        p = x.sub_(top).exp_()
        total = p.sum(3, keepdim=True)
        y = torch.matmul(p.div_(total).view(Hk, c * G, n), v).view(Hk, c, G, D)
        out[at:at + c] = y.transpose(0, 1).reshape(c, Hk * G, D)
        lse[at:at + c] = (top + total.log()).view(Hk, c, G).transpose(0, 1).reshape(c, Hk * G)
    return {"out": out, "lse": lse}


def _frequencies(case):
    """Radians per position of each pair, and what cosines and sines are multiplied by."""
    part, factor = case["part"], case["factor"]
    base = 10000.0 * factor ** (part / (part - 2)) if case["scaling"] == "base" else 10000.0
    w = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / part)
    gain = 1.0
    if case["scaling"] == "linear":
        w = w / factor
    elif case["scaling"] == "ramp":
        # fast pairs stay as they are, slow ones are stretched, between them a ramp over their turns
        keep = ((case["original"] * w / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        w = w * keep + w / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    return w, gain


def _angles(s):
    """Cosine and sine of every row's pairs, [rows, 1, part / 2]; angles in 64 bits."""
    case = s["case"]
    w, gain = _frequencies(case)
    starts, lens = s["starts"].long(), s["lens"].long()
    row = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(starts[1:], row, right=True)
    pos = lens[b] - starts[b + 1] + row
    angle = (pos[:, None].double() * w)[:, None, :]
    return b, pos, (angle.cos() * gain).float(), (angle.sin() * gain).float()


def _turned(x, cos, sin, case):
    x, part = x.float(), case["part"]
    if case["layout"] == "half":
        a, b = x[..., :part // 2], x[..., part // 2:part]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:part:2], x[..., 1:part:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., part:]], -1).to(_dtype(case))


def _plain_enter(s):
    case, pool, Hk, D = s["case"], s["pool"], s["case"]["kv_heads"], s["case"]["dim"]
    b, pos, cos, sin = _angles(s)
    page, t = s["table"].long()[b, pos // case["page"]], pos % 32
    block, e = pos % case["page"] // 32, 16 // pool.element_size()
    s["out"].copy_(_turned(s["q"], cos, sin, case))
    K = pool[:, :, 0].view(pool.shape[0], 1, Hk, case["page"] // 32, 2, D // e, 16, e)
    K[page, 0, :, block, t // 16, :, t % 16, :] = _turned(s["k"], cos, sin, case).unflatten(-1, (-1, e))
    if pool.dtype == torch.bfloat16:
        V = pool[:, :, 1].view(pool.shape[0], 1, Hk, case["page"] // 32, D, 4, 2, 4)
        V[page, 0, :, block, :, t % 16 // 4, t // 16, t % 4] = s["v"]
    else:
        V = pool[:, :, 1].view(pool.shape[0], 1, Hk, case["page"] // 32, 2, D, 4, 4)
        V[page, 0, :, block, t // 16, :, t % 16 // 4, t % 4] = s["v"]
    return {"q": s["out"], "pool": pool}


def _plain_rows(s):
    counts, page = s["counts"].long(), s["case"]["page"]
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), counts.cumsum(0)])
    row = torch.arange(s["sequence"].shape[0], device=DEV)
    b = torch.searchsorted(starts[1:], row, right=True)
    none = b == len(counts)
    b = b.clamp(max=len(counts) - 1)
    pos = torch.where(none, 0, s["lens"].long()[b] - starts[b + 1] + row)
    slot = s["table"].long()[b, pos // page] * page + pos % page
    return {"starts": starts.to(torch.int32), "sequence": torch.where(none, -1, b).to(torch.int32),
            "position": torch.where(none, -1, pos).to(torch.int32), "slot": torch.where(none, -1, slot).to(torch.int32)}


def _plain_score(s):
    logits, k, token = s["x"].float(), s["case"]["k"], s["token"].long()
    top = logits.amax(1, keepdim=True)
    x = logits - top
    e = x.exp()
    total = e.sum(1)
    lse = total.log()
    got = x.gather(1, token.clamp(min=0)[:, None])[:, 0] - lse
    out = {"logprob": torch.where(token < 0, 0.0, got), "entropy": lse - (e * x).sum(1) / total}
    if k:
        # the k largest, ties to the lowest token: logit and token make one whole number
        bits = logits.view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        at = (bits * 2**31 + (2**31 - 1 - torch.arange(x.shape[1], device=DEV))).topk(k, 1).indices
        out["top"], out["top_logprob"] = at.to(torch.int32), x.gather(1, at) - lse[:, None]
    return out


# -------------------------------------------------------- the library's calls


def _vs():
    root = os.path.join(os.getcwd(), "dart-pytorch_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import vector_store

    return vector_store


def _cache(s):
    """The cache over the state's pool, the sequences on it and the model's rotation, as a program keeps them."""
    if "cache" not in s:
        vs, case = _vs(), s["case"]
        if "pool" in s:
            s["cache"] = vs.PagedKVCache(s["pool"].shape[0], case["page"], case["kv_heads"], case["dim"],
                                         dtype=case["dtype"], memory=s["pool"])
        elif "table" in s:  # (the rows' places need the pages' numbers, not their contents)
            s["cache"] = vs.PagedKVCache(s["refs"].shape[0], case["page"], 1, 16)
        else:
            s["cache"] = vs.BeamSearch()
        if "table" in s:
            s["seqs"] = vs.KVSequences(s["table"], s["lens"], s["refs"])
        if case["kind"] == "enter":
            more = {"high": 32.0, "original": case["original"]} if case["scaling"] == "ramp" else {}
            s["rotary"] = vs.Rotary(case["dim"], dims=case["part"], base=10000.0, layout=case["layout"],
                                    scaling=case["scaling"], factor=case["factor"], **more)
    return s["cache"]


def _own_attend(s):
    case = s["case"]
    _cache(s).attend_rows(s["seqs"], s["q"], s["out"], starts=s["starts"], lse=s["lse"], causal=case["causal"],
                          window=case["window"], sinks=case["sinks"], stream=torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"], "lse": s["lse"]}


def _own_enter(s):
    cache = _cache(s)
    cache.append(s["seqs"], s["k"], s["v"], starts=s["starts"], rotary=s["rotary"], q=s["q"], q_out=s["out"],
                 stream=torch.cuda.current_stream().cuda_stream)
    return {"q": s["out"], "pool": s["pool"]}


def _own_rows(s):
    _cache(s).rows(s["seqs"], s["counts"], s["starts"], sequence=s["sequence"], position=s["position"],
                   slot=s["slot"], stream=torch.cuda.current_stream().cuda_stream)
    return {name: s[name] for name in ("starts", "sequence", "position", "slot")}


def _own_score(s):
    more = {"top_tokens": s["top"], "top_logprobs": s["top_logprob"]} if s["case"]["k"] else {}
    _cache(s).logprobs(s["x"], s["token"], s["logprob"], entropy=s["entropy"],
                       stream=torch.cuda.current_stream().cuda_stream, **more)
    out = {"logprob": s["logprob"], "entropy": s["entropy"]}
    return {**out, "top": s["top"], "top_logprob": s["top_logprob"]} if s["case"]["k"] else out


def run(s):
    if own:
        return {"attend": _own_attend, "enter": _own_enter, "rows": _own_rows, "score": _own_score}[s["case"]["kind"]](s)
    return {"attend": _plain_attend, "enter": _plain_enter, "rows": _plain_rows, "score": _plain_score}[s["case"]["kind"]](s)


# ------------------------------------------------------------- accounting


def work(case):
    if case["kind"] == "score":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (case["vocab"] * size + 12 + case["k"] * 8), "flops": 5.0 * case["rows"] * case["vocab"]}
    n, c = _sizes(case)
    if case["kind"] == "rows":
        pages = int((-(-n // case["page"]) - (n - c) // case["page"]).sum())  # entries that rows need
        return {"bytes": case["seqs"] * 12 + (int(c.sum()) + case["spare"]) * 12 + pages * 4, "flops": 0}
    size, H, Hk, D, R = 2 if case["dtype"] == "bf16" else 4, case["heads"], case["kv_heads"], case["dim"], int(c.sum())
    if case["kind"] == "enter":  # queries, keys and values in and out, 6 operations per rotated pair
        return {"bytes": R * 2 * (H + 2 * Hk) * D * size, "flops": 3.0 * R * (H + Hk) * case["part"]}
    seen = torch.zeros((), dtype=torch.float64)
    held = n.clone()
    if case["causal"]:
        first = n - c
        W, S = case["window"], case["sinks"]
        for a, b in zip(first.tolist(), n.tolist()):
            up = torch.arange(a + 1, b + 1, dtype=torch.float64)
            seen += (up.clamp(max=W) + (up - W).clamp(min=0, max=S)).sum() if W else up.sum()
        if W:
            low = (first + 1 - W).clamp(min=0)
            held = n - low + torch.clamp(low, max=S)
    else:
        seen += (n * c).sum()
    return {"bytes": int(held.sum()) * Hk * 2 * D * size + R * H * (2 * D * size + 4), "flops": 4.0 * float(seen) * H * D}


# ---------------------------------------------------------- 64-bit results


def _exact_attend(case, seed):
    s = prepare(case, seed)
    Hk, D, page, G = case["kv_heads"], case["dim"], case["page"], case["heads"] // case["kv_heads"]
    t = torch.arange(page)
    E = 16 // s["pool"].element_size()
    x = torch.arange(D)[None, :]
    block, h, g, i = (t // 32)[:, None], (t % 32 // 16)[:, None], (t % 16 // 4)[:, None], (t % 4)[:, None]
    # where each position and dimension of a page lies
    key = (block * 32 * D + ((h * (D // E) + x // E) * 16 + 4 * g + i) * E + x % E).to(DEV)
    value = (block * 32 * D + (((x * 4 + g) * 2 + h) * 4 + i if E == 8 else ((h * D + x) * 4 + g) * 4 + i)).to(DEV)
    out, lse = torch.empty(s["out"].shape, dtype=torch.float64, device=DEV), torch.empty(s["lse"].shape, dtype=torch.float64, device=DEV)
    for b, (n, c, at) in enumerate(zip(*s["sizes"])):
        ids = s["table"][b, :-(-n // page)].long()
        for kv in range(Hk):
            K = s["pool"][ids, 0, 0, kv][:, key].reshape(-1, D)[:n].double()
            V = s["pool"][ids, 0, 1, kv][:, value].reshape(-1, D)[:n].double()
            for r in range(0, c, 2048):
                m = min(2048, c - r)
                q = s["q"][at + r:at + r + m, kv * G:kv * G + G].double().reshape(m * G, D)
                y = (q @ K.T) * D ** -0.5
                if case["causal"]:
                    last = torch.arange(n - c + r, n - c + r + m, device=DEV).repeat_interleave(G)[:, None]
                    p = torch.arange(n, device=DEV)[None, :]
                    seen = p <= last
                    if case["window"]:
                        seen &= (p > last - case["window"]) | (p < case["sinks"])
                    y = torch.where(seen, y, -math.inf)
                z = torch.logsumexp(y, 1, keepdim=True)
                out[at + r:at + r + m, kv * G:kv * G + G] = ((y - z).exp() @ V).view(m, G, D)
                lse[at + r:at + r + m, kv * G:kv * G + G] = z.view(m, G)
    return {"out": out, "lse": lse}


def _exact_enter(case, seed):
    s = prepare(case, seed)
    w, gain = _frequencies(case)
    part, D, Hk, page, pool = case["part"], case["dim"], case["kv_heads"], case["page"], s["pool"].double()
    E, x = 16 // s["pool"].element_size(), torch.arange(D, device=DEV)
    q = s["q"].double().clone()
    first, second = (torch.arange(part // 2), torch.arange(part // 2) + part // 2) if case["layout"] == "half" else \
        (torch.arange(0, part, 2), torch.arange(1, part, 2))
    for b, (n, c, at) in enumerate(zip(*s["sizes"])):
        pos = torch.arange(n - c, n, device=DEV)
        turn = torch.polar(torch.full((), gain, dtype=torch.float64, device=DEV), pos[:, None].double() * w)[:, None, :]
        k, v = s["k"][at:at + c].double().clone(), s["v"][at:at + c].double()
        for y in (q[at:at + c], k):
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
        ids, off, t = s["table"][b].long()[pos // page], pos % page // 32 * 32 * D, pos % 32
        h, g, i = (t // 16)[:, None], (t % 16 // 4)[:, None], (t % 4)[:, None]
        key = off[:, None] + ((h * (D // E) + x // E) * 16 + 4 * g + i) * E + x % E
        value = off[:, None] + (((x * 4 + g) * 2 + h) * 4 + i if E == 8 else ((h * D + x) * 4 + g) * 4 + i)
        heads = torch.arange(Hk, device=DEV)[None, :, None]
        pool[ids[:, None, None], 0, 0, heads, key[:, None, :]] = k
        pool[ids[:, None, None], 0, 1, heads, value[:, None, :]] = v
    return {"q": q, "pool": pool}


def _exact_score(case, seed):
    s = prepare(case, seed)
    logprob, entropy, tops = [], [], []
    for x, token in zip(s["x"].split(256), s["token"].long().split(256)):
        logp = torch.log_softmax(x.double(), 1)
        got = logp.gather(1, token.clamp(min=0)[:, None])[:, 0]
        logprob.append(torch.where(token < 0, 0.0, got))
        entropy.append(-(logp.exp() * logp).sum(1))
        if case["k"]:
            tops.append(logp.topk(case["k"], 1).values)
    out = {"logprob": torch.cat(logprob), "entropy": torch.cat(entropy)}
    return {**out, "top": None, "top_logprob": torch.cat(tops)} if case["k"] else out


def exact(case, seed):
    if case["kind"] == "rows":
        return None  # whole numbers: nothing is rounded
    return {"attend": _exact_attend, "enter": _exact_enter, "score": _exact_score}[case["kind"]](case, seed)
