"""Rotary positions in large calls: several heads that share their angles, by themselves and on the way into the cache.
How many go together follows from the sizes; the rules stand here again, so that no case drifts off them."""
import re

import numpy as np
import pytest

import _decode as D
import _prompt as P
from test_gpu_attend import View
from test_gpu_rotary import Entered, check, host

pytestmark = pytest.mark.gpu


def cus(vs):
    return int(re.search(r"(\d+) CUs", vs.device_name(0)).group(1))


def threads_per_unit(vs, rows, heads, dim, dims, dtype, pieces, in_place):
    """Over how many threads a unit's heads are spread."""
    e = 8 if dtype == "bf16" else 4
    units = dims // 2 // (e if pieces else 1) + (0 if in_place else (dim - dims) // (e if pieces else 1))
    spread = heads
    while spread > 1 and rows * units * (spread // 2) >= cus(vs) * 1024:
        spread = (spread + 1) // 2
    return spread


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,rows,heads,dim,dims,offset,spread", [
    ("bf16", 6000, 13, 128, 128, 0, 7), ("f32", 4000, 13, 128, 128, 0, 7), ("bf16", 4000, 12, 128, 64, 0, 6),
    ("f32", 5000, 7, 96, 32, 0, 4), ("bf16", 4001, 13, 64, 64, 1, 4), ("f32", 3001, 5, 80, 20, 1, 3), ("bf16", 5003, 3, 128, 94, 0, 1),
])
def test_rows(vs, layout, dtype, rows, heads, dim, dims, offset, spread):
    """Forward, backward and in place; rows that start anywhere; what is not turned is copied."""
    A, rng = vs.DeviceArray, np.random.default_rng(rows)
    e = 8 if dtype == "bf16" else 4
    wide = heads * dim + 3 * offset
    pieces = offset == 0 and dims % (2 * e) == 0
    assert threads_per_unit(vs, rows, heads, dim, dims, dtype, pieces, False) == spread < heads
    b, x = D.stored(rng.standard_normal((rows, wide)), dtype)
    part = lambda a: a[:, offset:offset + heads * dim].reshape(rows, heads, dim)  # noqa: E731
    view = lambda a: View(a, (rows, heads, dim), (wide, dim, 1), offset)  # noqa: E731
    rest = [i for i in range(wide) if not offset <= i < offset + heads * dim]
    pos = rng.integers(0, 100000, rows)
    at, rot = A.of(pos, "i32"), vs.Rotary(dim, dims=dims, layout=layout, gain=1.25)
    src = A.of(b, dtype)
    for backward in (False, True):
        out = A.of(np.zeros_like(b), dtype)
        rot.rotate(view(src), view(out), at, backward=backward)
        got = host(out, dtype)
        check(part(got), part(x), pos, rot, dtype, backward)
        assert np.array_equal(part(got)[..., dims:], part(x)[..., dims:]) and not got[:, rest].any()
        assert np.array_equal(src.numpy(), b)
        same = A.of(b, dtype)
        rot.rotate(view(same), view(same), at, backward=backward)
        assert np.array_equal(part(host(same, dtype)), part(got)) and np.array_equal(same.numpy()[:, rest], b[:, rest])
    rot.close()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,dim,dims,heads,kv", [("bf16", 64, 64, 5, 5), ("f32", 64, 64, 17, 2), ("bf16", 80, 20, 17, 2),
                                                    ("bf16", 128, 32, 18, 3), ("f32", 48, 46, 4, 6)])
def test_rows_enter_the_cache_turned(vs, layout, dtype, dim, dims, heads, kv):
    """Four query heads share their angles; the last set of them is not full."""
    A = vs.DeviceArray
    e = Entered(vs, [1700, 33, 2500], [1500, 33, 1400], heads, kv, dim, 64, dtype)
    rows = len(e.pos)
    assert (rows // 32 + 2 * 3 + 1) * (kv + heads // 4) >= 2 * cus(vs)
    rot = vs.Rotary(dim, dims=dims, layout=layout, gain=1.1)
    k, v, q, out, starts = A.of(e.kb, dtype), A.of(e.vb, dtype), A.of(e.qb, dtype), A(e.q.shape, dtype), A.of(e.starts, "i32")
    e.cache.append(e.seqs, k, v, starts=starts, rotary=rot, q=q, q_out=out)
    e.cache.check()
    e.compare(rot, out)
    e.cache.append(e.seqs, k, v, starts=starts, rotary=rot, q=q, q_out=q)  # in place
    assert np.array_equal(q.numpy(), out.numpy())
    e.cache.close()
    rot.close()


def test_more_blocks_than_one_pass_of_the_grid(vs):
    """Past 2^20 workgroups: 540,000 sequences of one row, a key-value head and a query head each."""
    A, rng, n, dim = vs.DeviceArray, np.random.default_rng(8), 540_000, 16
    lens = 1 + np.arange(n) % 32
    mem = A((n, 2, 32 * dim), "bf16")
    cache = vs.PagedKVCache(n, 32, 1, dim, memory=mem)
    seqs = vs.KVSequences(A.of(rng.permutation(n)[:, None], "i32"), A.of(lens, "i32"), A.of(np.ones(n), "i32"))
    rot = vs.Rotary(dim)
    (kb, k), (vb, _), (qb, q) = (D.stored(rng.standard_normal((n, 1, dim)), "bf16") for _ in range(3))
    out = A((n, 1, dim), "bf16")
    cache.append(seqs, A.of(kb, "bf16"), A.of(vb, "bf16"), rotary=rot, q=A.of(qb, "bf16"), q_out=out)
    cache.check()
    kp, vp = D.places(dim, "bf16")
    pages, pool = seqs.table.numpy()[:, 0], mem.numpy()
    at = lens - 1
    assert np.array_equal(pool[pages[:, None], 1, vp[at]], vb[:, 0])
    got_k = D.from_bf16(pool[pages[:, None], 0, kp[at]])
    angle = at[:, None] * rot.frequencies
    c, s = np.cos(angle), np.sin(angle)
    for got, x in ((got_k, k[:, 0]), (D.from_bf16(out.numpy())[:, 0], q[:, 0])):
        a, b = x[:, :8].astype(np.float64), x[:, 8:].astype(np.float64)
        want = np.concatenate([a * c - b * s, b * c + a * s], 1)
        size = np.tile(np.abs(a) + np.abs(b), 2)
        D.assert_rounded(got, want, P.turn_tolerance(size, at, rot.frequencies), "bf16")
    cache.close()
    rot.close()
