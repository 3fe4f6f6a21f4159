"""Rotary positions against their formula in 64 bits: by themselves, backwards, and
on the way into the paged cache."""
import numpy as np
import pytest

import _decode as D
import _prompt as P
from _hip import Stream
from test_gpu_attend import View

pytestmark = pytest.mark.gpu


def host(t, dtype):
    a = t.numpy()
    return D.from_bf16(a) if dtype == "bf16" else a


def check(got, x, positions, rot, dtype, backward=False):
    want, size = P.turned(x.astype(np.float64), positions, rot.frequencies, rot.gain, rot.layout, backward)
    off = P.turn_tolerance(size, positions, rot.frequencies)
    off[..., rot.dims:] = 0
    D.assert_rounded(got, want, off, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,dims", [(64, 64), (128, 128), (256, 64), (80, 20), (48, 6), (16, 2), (96, 94), (7, 4), (33, 16), (512, 512)])
def test_rows(vs, dtype, layout, dim, dims):
    A, rng = vs.DeviceArray, np.random.default_rng(dim)
    rot = vs.Rotary(dim, dims=dims, layout=layout)
    for rows, heads in ((1, 1), (3, 5), (70, 12), (300, 1), (0, 4)):
        b, x = D.stored(rng.standard_normal((rows, heads, dim)), dtype)
        pos = rng.integers(0, 5000, rows)
        out, src, at = A((rows, heads, dim), dtype), A.of(b, dtype), A.of(pos, "i32")
        rot.rotate(src, out, at)
        got = host(out, dtype)
        check(got, x, pos, rot, dtype)
        assert np.array_equal(src.numpy(), b)
        rot.rotate(src, src, at)  # in place
        assert np.array_equal(host(src, dtype), got)
    rot.close()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_negative_positions(vs, layout):
    """Angles lose nothing: 2^31 - 1 positions of one radian are as exact as the first ones."""
    A, rng = vs.DeviceArray, np.random.default_rng(1)
    rot = vs.Rotary(64, layout=layout)
    pos = np.concatenate([[0, 1, -1, 2**31 - 1, -2**31, 2**24 + 1, 2**24 - 1], rng.integers(-2**31, 2**31, 200)])
    b, x = D.stored(rng.standard_normal((len(pos), 2, 64)), "f32")
    out = A(x.shape, "f32")
    rot.rotate(A.of(b, "f32"), out, A.of(pos, "i32"))
    check(out.numpy(), x, pos, rot, "f32")


def test_quarter_turns_are_exact_enough(vs):
    """Frequencies that land on the octants' borders."""
    A = vs.DeviceArray
    w = np.array([2 * np.pi / 8, 2 * np.pi / 4, -2 * np.pi / 3, 0.0])
    rot = vs.Rotary(8, frequencies=w)
    pos = np.arange(-40, 40)
    x = np.tile(np.array([1, 1, 1, 1, 0, 0, 0, 0], np.float32), (80, 1, 1))
    out = A(x.shape, "f32")
    rot.rotate(A.of(x, "f32"), out, A.of(pos, "i32"))
    check(out.numpy(), x, pos, rot, "f32")
    assert np.array_equal(out.numpy()[:, 0, [3, 7]], x[:, 0, [3, 7]])  # a pair that does not turn


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                dict(scaling="ramp", factor=8.0, original=512),
                                dict(scaling="ramp", factor=32.0, original=2048, low=1.0, high=32.0, ramp_by="index"),
                                dict(base=500000.0), dict(gain=0.5)])
def test_scalings(vs, kw):
    A, rng = vs.DeviceArray, np.random.default_rng(2)
    dims, rot = 64, vs.Rotary(64, **kw)
    base, factor = kw.get("base", 10000.0), kw.get("factor", 1.0)
    if kw.get("scaling") == "base":
        base *= factor ** (dims / (dims - 2))
    w = np.array([base ** (-2 * i / dims) for i in range(dims // 2)])
    if kw.get("scaling") == "linear":
        w = w / factor
    if kw.get("scaling") == "ramp":
        low, high, orig = kw.get("low", 1.0), kw.get("high", 4.0), kw["original"]
        turns = orig * w / (2 * np.pi)
        if kw.get("ramp_by") == "index":
            first = np.floor(32 * np.log(orig / (high * 2 * np.pi)) / np.log(base))
            last = np.ceil(32 * np.log(orig / (low * 2 * np.pi)) / np.log(base))
            keep = 1 - np.clip((np.arange(32) - first) / (last - first), 0, 1)
        else:
            keep = np.clip((turns - low) / (high - low), 0, 1)
        assert (keep[:3] == 1).all() and (keep[-3:] == 0).all() and ((keep > 0) & (keep < 1)).any()
        w = keep * w + (1 - keep) * w / factor
        assert rot.gain == pytest.approx(0.1 * np.log(factor) + 1)
    np.testing.assert_allclose(rot.frequencies, w, rtol=1e-12)
    pos = rng.integers(0, 60000, 50)
    b, x = D.stored(rng.standard_normal((50, 3, 64)), "f32")
    out = A(x.shape, "f32")
    rot.rotate(A.of(b, "f32"), out, A.of(pos, "i32"))
    check(out.numpy(), x, pos, rot, "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_is_the_gradient(vs, layout, dtype):
    """Against the formula's, and against differences: the turn is linear, so a difference of any size is exact but
    for rounding."""
    A, rng = vs.DeviceArray, np.random.default_rng(3)
    rows, heads, dim = 20, 3, 32
    rot = vs.Rotary(dim, dims=24, layout=layout, gain=1.25)
    pos = A.of(rng.integers(0, 3000, rows), "i32")
    gb, g = D.stored(rng.standard_normal((rows, heads, dim)), dtype)
    back = A(g.shape, dtype)
    rot.rotate(A.of(gb, dtype), back, pos, backward=True)
    dx = host(back, dtype)
    check(dx, g, pos.numpy(), rot, dtype, backward=True)
    if dtype == "f32":  # d (g . y(x)) / dx_j, for every row and head at once
        y = A(g.shape, "f32")
        for j in range(dim):
            x = np.zeros(g.shape, np.float32)
            x[..., j] = 1
            rot.rotate(A.of(x, "f32"), y, pos)
            diff = (y.numpy().astype(np.float64) * g).sum(-1)  # (y of 0 is 0)
            # two products of one rounding each, and the gradient's own few
            np.testing.assert_allclose(dx[..., j], diff, rtol=0, atol=1.25 * 2 * np.abs(g).max() * 16 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strided_rows_in_place(vs, dtype, offset):
    """Queries as a part of a projection's output, turned where they lie."""
    A, rng = vs.DeviceArray, np.random.default_rng(4)
    rows, heads, dim, wide = 40, 4, 32, 4 * 32 + 40 + offset
    b, x = D.stored(rng.standard_normal((rows, wide)), dtype)
    base, pos = A.of(b, dtype), rng.integers(0, 100, rows)
    rot = vs.Rotary(dim)
    view = View(base, (rows, heads, dim), (wide, dim, 1), offset)
    rot.rotate(view, view, A.of(pos, "i32"))
    got = base.numpy()
    assert np.array_equal(np.delete(got, np.s_[offset:offset + 128], 1), np.delete(b, np.s_[offset:offset + 128], 1))
    part = (D.from_bf16(got) if dtype == "bf16" else got)[:, offset:offset + 128].reshape(rows, heads, dim)
    check(part, x[:, offset:offset + 128].reshape(rows, heads, dim), pos, rot, dtype)


class Entered:
    """A cache on which counts[b] rows enter at the end of sequence b."""

    def __init__(self, vs, lens, counts, heads, kv, dim, page=32, dtype="bf16", seed=0):
        A, rng = vs.DeviceArray, np.random.default_rng(seed)
        self.vs, self.lens, self.counts, self.dtype = vs, lens, counts, dtype
        held = [-(-n // page) for n in lens]
        npages = sum(held) + 2
        self.table = np.full((len(lens), max(held + [1])), -1, np.int32)
        ids = rng.permutation(npages)
        at = 0
        for b, h in enumerate(held):
            self.table[b, :h] = ids[at:at + h]
            at += h
        refs = np.bincount(self.table[self.table >= 0], minlength=npages)
        self.cache = vs.PagedKVCache(npages, page, kv, dim, dtype=dtype)
        self.seqs = vs.KVSequences(A.of(self.table, "i32"), A.of(lens, "i32"), A.of(refs, "i32"))
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        rows = int(self.starts[-1])
        (self.qb, self.q), (self.kb, self.k), (self.vb, self.v) = (
            D.stored(rng.standard_normal((rows, h, dim)), dtype) for h in (heads, kv, kv))
        self.pos = np.concatenate([np.arange(n - c, n) for n, c in zip(lens, counts)] + [np.zeros(0, int)])

    def held(self, b):
        """The keys and values of sequence b's new positions."""
        A, n, c = self.vs.DeviceArray, self.lens[b], self.counts[b]
        k, v = A((c, self.cache.kv_heads, self.cache.head_dim), self.dtype), A((c, self.cache.kv_heads, self.cache.head_dim), self.dtype)
        self.cache.read(self.seqs, b, n - c, k, v)
        return host(k, self.dtype), v.numpy()

    def compare(self, rot, q_out):
        check(host(q_out, self.dtype), self.q, self.pos, rot, self.dtype)
        for b, c in enumerate(self.counts):
            if c:
                at = slice(self.starts[b], self.starts[b + 1])
                k, v = self.held(b)
                check(k, self.k[at], self.pos[at], rot, self.dtype)
                assert np.array_equal(v, self.vb[at])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,dims,heads,kv", [(64, 64, 8, 2), (128, 128, 5, 5), (80, 20, 3, 1), (96, 48, 17, 1), (256, 2, 2, 2)])
def test_rows_enter_the_cache_turned(vs, dtype, layout, dim, dims, heads, kv):
    A = vs.DeviceArray
    e = Entered(vs, [40, 1, 200, 33, 64, 5000], [7, 1, 150, 0, 64, 70], heads, kv, dim, 32, dtype)
    rot = vs.Rotary(dim, dims=dims, layout=layout, gain=1.1)
    q, out = A.of(e.qb, dtype), A(e.q.shape, dtype)
    e.cache.append(e.seqs, A.of(e.kb, dtype), A.of(e.vb, dtype), starts=A.of(e.starts, "i32"), rotary=rot, q=q, q_out=out)
    e.cache.check()
    e.compare(rot, out)
    e.cache.append(e.seqs, A.of(e.kb, dtype), A.of(e.vb, dtype), starts=A.of(e.starts, "i32"), rotary=rot, q=q, q_out=q)
    assert np.array_equal(q.numpy(), out.numpy())  # in place


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_row_each(vs, dtype):
    A = vs.DeviceArray
    e = Entered(vs, [1, 32, 33, 700, 64], [1] * 5, 4, 2, 64, 32, dtype)
    rot, out = vs.Rotary(64), A(e.q.shape, dtype)
    e.cache.append(e.seqs, A.of(e.kb, dtype), A.of(e.vb, dtype), rotary=rot, q=A.of(e.qb, dtype), q_out=out)
    e.compare(rot, out)
    e.cache.append(e.seqs, A.of(e.kb, dtype), A.of(e.vb, dtype), rotary=rot)  # keys alone
    e.compare(rot, out)


def test_parts_of_a_projection(vs):
    """Queries, keys and values side by side in a row; the queries turned where they lie."""
    A = vs.DeviceArray
    e = Entered(vs, [40, 90], [30, 90], 4, 2, 32, 32, "bf16")
    rows, rot = len(e.pos), vs.Rotary(32)
    base = A.of(np.concatenate([e.qb, e.kb, e.vb], 1), "bf16")
    part = lambda h0, h: View(base, (rows, h, 32), (8 * 32, 32, 1), h0 * 32)  # noqa: E731
    e.cache.append(e.seqs, part(4, 2), part(6, 2), starts=A.of(e.starts, "i32"), rotary=rot, q=part(0, 4), q_out=part(0, 4))
    got = base.numpy()
    assert np.array_equal(got[:, 4:], np.concatenate([e.kb, e.vb], 1))
    out = A.of(np.ascontiguousarray(got[:, :4]), "bf16")
    e.compare(rot, out)


def test_what_has_no_place(vs):
    """Missing pages and positions below 0: nothing is stored, queries are turned all the same; rows behind the last
    sequence's are left as they were, and so is the cache behind an extend that did not fit."""
    A = vs.DeviceArray
    e = Entered(vs, [40, 70], [40, 70], 2, 1, 32, 32, "f32")
    e.table[1, 1] = -1
    seqs = vs.KVSequences(A.of(e.table, "i32"), A.of([30, 70], "i32"), e.seqs.refs)  # 10 rows of the first are before it
    pos = np.concatenate([np.arange(-10, 30), np.arange(70)])
    rot, out = vs.Rotary(32), A.of(np.full((115, 2, 32), 7.0), "f32")
    pad = lambda x: A.of(np.concatenate([x, np.full((5,) + x.shape[1:], 3, x.dtype)]), "f32")  # noqa: E731
    e.cache.append(seqs, pad(e.kb), pad(e.vb), starts=A.of([0, 40, 110], "i32"), rotary=rot, q=pad(e.qb), q_out=out)
    e.cache.check()
    got = out.numpy()
    check(got[:110], e.q, pos, rot, "f32")
    assert (got[110:] == 7).all()
    k, v = A((70, 1, 32), "f32"), A((70, 1, 32), "f32")
    e.cache.read(e.seqs, 1, 0, k, v)
    check(k.numpy()[:32], e.k[40:72], np.arange(32), rot, "f32")
    check(k.numpy()[64:], e.k[104:], np.arange(64, 70), rot, "f32")


def test_nothing_is_stored_behind_an_extend_that_did_not_fit(vs):
    A, rng = vs.DeviceArray, np.random.default_rng(5)
    cache, rot = vs.PagedKVCache(3, 32, 1, 32, dtype="f32"), vs.Rotary(32)
    seqs = cache.new_sequences(1, 8)
    k, v, q = (rng.standard_normal((90, 1, 32)).astype(np.float32) for _ in range(3))
    starts, qd, out = A.of([0, 90], "i32"), A.of(q, "f32"), A(q.shape, "f32")
    cache.extend(seqs, 90)
    cache.append(seqs, A.of(k, "f32"), A.of(v, "f32"), starts=starts, rotary=rot)
    cache.extend(seqs, 40)
    cache.append(seqs, A.of(v, "f32"), A.of(k, "f32"), starts=starts, rotary=rot, q=qd, q_out=out)
    with pytest.raises(vs.VsError, match="pages short"):
        cache.check()
    check(out.numpy(), q, np.arange(90), rot, "f32")
    kk, vv = A(k.shape, "f32"), A(k.shape, "f32")
    cache.read(seqs, 0, 0, kk, vv)
    check(kk.numpy(), k, np.arange(90), rot, "f32")
    assert np.array_equal(vv.numpy(), v)


def test_streams_and_graphs(vs):
    A = vs.DeviceArray
    e = Entered(vs, [300, 40], [200, 40], 8, 2, 64, 32, "bf16")
    rot, st = vs.Rotary(64), Stream()
    q, k, v, starts, out = A.of(e.qb, "bf16"), A.of(e.kb, "bf16"), A.of(e.vb, "bf16"), A.of(e.starts, "i32"), A(e.q.shape, "bf16")
    st.begin()
    e.cache.append(e.seqs, k, v, starts=starts, rotary=rot, q=q, q_out=out, stream=st.ptr)
    graph = st.end()
    for i in range(3):
        out.upload(np.zeros_like(e.qb))
        st.replay(graph)
        e.compare(rot, out)
        e.cache.append(e.seqs, v, k, starts=starts, rotary=rot)  # (the program's own work between the replays)


def test_refusals(vs):
    A = vs.DeviceArray
    for kw in (dict(dims=3), dict(dims=0), dict(dims=66), dict(layout="other"), dict(scaling="other"), dict(base=0.5),
               dict(factor=0.0), dict(scaling="ramp"), dict(scaling="ramp", original=100, low=4, high=2),
               dict(scaling="ramp", original=100, ramp_by="other"), dict(frequencies=np.ones(5)),
               dict(frequencies=np.full(32, np.nan)), dict(gain=float("inf"))):
        with pytest.raises(ValueError):
            vs.Rotary(64, **kw)
    rot = vs.Rotary(64)
    x, pos = A((6, 2, 64), "f32"), A.of(np.zeros(6), "i32")
    for a, b, p in ((A((6, 2, 32), "f32"), x, pos), (x, A((6, 2, 64), "bf16"), pos), (x, x, A.of(np.zeros(5), "i32")),
                    (x, View(x, (6, 2, 64), (128, 64, 1), 4), pos), (A((6, 2, 64), "i32"), A((6, 2, 64), "i32"), pos)):
        with pytest.raises(ValueError):
            rot.rotate(a, b, p)
    e = Entered(vs, [40], [40], 2, 1, 32, 32, "bf16")
    k, v, q, starts = A.of(e.kb, "bf16"), A.of(e.vb, "bf16"), A.of(e.qb, "bf16"), A.of(e.starts, "i32")
    small = vs.Rotary(32)
    for kw in (dict(rotary=rot), dict(rotary=small, q=q), dict(q=q, q_out=q), dict(rotary=small, q_out=q),
               dict(rotary=small, q=k, q_out=k), dict(rotary=small, q=q, q_out=A((40, 2, 16), "bf16")),
               dict(rotary=small, q=q, q_out=View(q, (40, 2, 32), (64, 32, 1), 2))):
        with pytest.raises(ValueError):
            e.cache.append(e.seqs, k, v, starts=starts, **kw)


@pytest.mark.parametrize("pad", [0, 24])
def test_parts_of_a_head_turned_in_place(vs, pad):
    """Queries, keys and values side by side in each head, [rows, heads, 3, dim]: they share no byte, so the queries are
    turned where they lie."""
    A, heads, dim = vs.DeviceArray, 3, 32
    e = Entered(vs, [40, 90], [30, 90], heads, heads, dim, 32, "bf16")
    rows, rot, wide = len(e.pos), vs.Rotary(dim), heads * 3 * dim + pad
    host = np.zeros((rows, wide), np.uint16)
    host[:, :wide - pad] = np.stack([e.qb, e.kb, e.vb], 2).reshape(rows, -1)
    base = A.of(host, "bf16")
    part = lambda i: View(base, (rows, heads, dim), (wide, 3 * dim, 1), i * dim)  # noqa: E731
    e.cache.append(e.seqs, part(1), part(2), starts=A.of(e.starts, "i32"), rotary=rot, q=part(0), q_out=part(0))
    got = base.numpy()[:, :wide - pad].reshape(rows, heads, 3, dim)
    assert np.array_equal(got[:, :, 1:], np.stack([e.kb, e.vb], 2))
    e.compare(rot, A.of(np.ascontiguousarray(got[:, :, 0]), "bf16"))
    with pytest.raises(ValueError, match="overlaps k or v"):
        e.cache.append(e.seqs, part(1), part(2), starts=A.of(e.starts, "i32"), rotary=rot, q=A.of(e.qb, "bf16"), q_out=part(1))


def test_strides_past_all_memory(vs):
    """Strides of so many rows that no address holds their sum are refused before it is taken."""
    A = vs.DeviceArray
    base, rot, n = A((4, 1, 64), "f32"), vs.Rotary(64), 2**31 - 2000
    far = View(base, (n, 1, 64), (2**40, 64, 1))
    near = View(base, (n, 1, 64), (64, 64, 1))
    for x, out in ((far, near), (near, far), (far, far)):
        with pytest.raises(ValueError, match="stride"):
            rot.rotate(x, out, View(A((4,), "i32"), (n,), (1,)))
    e = Entered(vs, [40], [40], 1, 1, 64, 32, "f32")
    starts = A.of(e.starts, "i32")
    with pytest.raises(ValueError, match="stride"):
        e.cache.append(e.seqs, near, near, starts=starts, rotary=rot, q=near, q_out=far)
    with pytest.raises(ValueError, match="stride"):
        e.cache.attend_rows(e.seqs, near, far, starts=starts)
