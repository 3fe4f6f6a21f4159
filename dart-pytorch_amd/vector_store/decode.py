"""Decoding on the GPU that holds the index: a paged key-value cache with the
attention of one new token or of many, rotary positions, beam search and log
probabilities.

The reference's vector store has no counterpart.  A program retrieves passages
with an index of this package and lets a model answer with them; these are the
model's steps that read what stays resident in HBM: the cache of keys and
values, and the choice of the next tokens.

  cache = PagedKVCache(pages, 32, kv_heads, head_dim, layers=layers)
  seqs, spare = cache.new_sequences(beams, width), cache.new_sequences(beams, width, seqs.refs)
  beams = BeamSearch()
  per token:
    cache.extend(seqs, 1)                        # a position for the new token
    per layer: cache.attend(seqs, q, out, k=k, v=v, layer=i)
    beams.select(logits, scores, next_scores, tokens, parents)
    beams.reorder(parents, history, next_history, tail=tokens)
    cache.fork(seqs, parents, spare); seqs, spare = spare, seqs
  now and then, and before the tokens are used:
    cache.check()                                # raises what did not fit; the cache is whole then

A prompt enters in chunks of any size, beside requests that decode:

  rotary = Rotary(head_dim)
  per chunk:
    cache.extend(seqs, counts)                   # how many rows each sequence brings
    cache.rows(seqs, counts, starts, position=positions)
    per layer:
      cache.append(seqs, k, v, starts=starts, layer=i, rotary=rotary, q=q, q_out=q)
      cache.attend_rows(seqs, q, out, starts=starts, layer=i)
    beams.logprobs(logits, tokens, out)          # where given tokens are scored

Buffers are anything in device memory with data_ptr(), shape, stride() and
dtype: DeviceArray of this module or a tensor of a framework that works on the
same GPU (imported before this package loads its library, so that both use the
HIP runtime that the framework brings).  Where a buffer says where it lies
(get_device(), -1 for host memory) it has to be the handle's device.  Calls run
on `stream` (an integer hipStream_t, 0 the default stream) and return without
waiting for it.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _native as N

_CODES = {"f32": N.VS_DTYPE_F32, "float32": N.VS_DTYPE_F32, "bf16": N.VS_DTYPE_BF16,
          "bfloat16": N.VS_DTYPE_BF16, "i32": -4, "int32": -4, "u8": -1, "uint8": -1, "bool": -1}
_SIZES = {N.VS_DTYPE_F32: 4, N.VS_DTYPE_BF16: 2, -4: 4, -1: 1}
_SEEN: dict = {}  # dtype objects already looked up
_I32, _U8 = -4, -1


def _code(dtype) -> int:
    c = _SEEN.get(dtype)
    if c is None:
        c = _CODES.get(str(dtype).rpartition(".")[2])
        if c is None:
            raise ValueError(f"unsupported element type {dtype}")
        _SEEN[dtype] = c
    return c


class DeviceArray:
    """A contiguous array in device memory that this package allocated.

    dtype: "f32", "bf16" (numpy: uint16 bit patterns), "i32" or "u8"."""

    _NUMPY = {N.VS_DTYPE_F32: np.float32, N.VS_DTYPE_BF16: np.uint16, _I32: np.int32, _U8: np.uint8}

    def __init__(self, shape, dtype: str = "f32", device: int = 0):
        self.shape = tuple(int(s) for s in shape)
        if any(s < 0 for s in self.shape):
            raise ValueError(f"negative size in {self.shape}")
        self.dtype = dtype
        self.device = int(device)
        self._code = _code(dtype)
        out, s = [], 1
        for n in reversed(self.shape):
            out.append(s)
            s *= n
        self._stride = tuple(reversed(out))
        self.buf = N.DeviceBuffer(max(1, math.prod(self.shape)) * _SIZES[self._code], device)

    @classmethod
    def of(cls, a, dtype: str, device: int = 0) -> "DeviceArray":
        d = cls(np.shape(a), dtype, device)
        d.upload(a)
        return d

    def data_ptr(self) -> int:
        return self.buf.ptr.value

    def stride(self):
        return self._stride

    def is_contiguous(self) -> bool:
        return True

    def get_device(self) -> int:
        return self.device

    def upload(self, a) -> "DeviceArray":
        a = np.ascontiguousarray(a, self._NUMPY[self._code])
        if a.shape != self.shape:
            raise ValueError(f"shape {a.shape}, expected {self.shape}")
        if a.size:
            self.buf.upload(a)
        return self

    def numpy(self) -> np.ndarray:
        """A host copy (waits for the default stream's work, not for other streams')."""
        out = np.empty(self.shape, self._NUMPY[self._code])
        if out.size:
            self.buf.download(out)
        return out


# A decoding step of a small model is a few microseconds on the GPU, so the
# checks below take the straight way where all is well.


def _device_of(t):
    """The device that a buffer says it lies on; None if it does not say."""
    try:
        return t.get_device()
    except AttributeError:
        return None


def _on(t, what, device) -> None:
    try:
        on = t.get_device()
    except AttributeError:
        return
    if on != device:
        raise ValueError(f"{what}: in {'host memory' if on < 0 else f'memory of device {on}'}, expected device {device}")


def _rows(t, what, shape, code, device=None):
    """Pointer and strides of a buffer of `shape` whose last dimension is contiguous (on `device`, if given)."""
    if device is not None:
        _on(t, what, device)
    st = t.stride()
    if t.shape != shape or _SEEN.get(t.dtype) != code or st[-1] != 1:
        if _code(t.dtype) != code:
            raise ValueError(f"{what}: element type {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")
        if st[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{what}: the last dimension is not contiguous")
    return t.data_ptr(), st


def _flat(t, what, shape, code, device=None) -> int:
    """Pointer of a contiguous buffer of `shape` (on `device`, if given)."""
    if device is not None:
        _on(t, what, device)
    try:
        fine = t.is_contiguous() and t.shape == shape and _SEEN.get(t.dtype) == code
    except AttributeError:
        fine = False
    if not fine:
        _look_closely(t, what, shape, code)
    return t.data_ptr()


def _look_closely(t, what, shape, code) -> None:
    if _code(t.dtype) != code:
        raise ValueError(f"{what}: element type {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")
    n = 1
    for size, s in zip(shape[::-1], t.stride()[::-1]):
        if s != n and size > 1:
            raise ValueError(f"{what}: not contiguous")
        n *= size


def _list(t, what, n, code, device=None) -> int:
    """Pointer of a contiguous buffer of n elements, whatever its shape (on `device`, if given)."""
    if device is not None:
        _on(t, what, device)
    shape = t.shape
    if len(shape) == 2 and shape[0] * shape[1] == n:  # (beams' outputs, [requests, k])
        try:
            fine = t.is_contiguous() and _SEEN.get(t.dtype) == code
        except AttributeError:
            fine = False
        if not fine:
            _look_closely(t, what, tuple(shape), code)
        return t.data_ptr()
    if math.prod(shape) != n:
        raise ValueError(f"{what}: shape {tuple(shape)}, expected {n} elements")
    return _flat(t, what, tuple(shape), code)


class _SeqsC(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("refs", ctypes.c_void_p),
                ("nseq", ctypes.c_int64), ("width", ctypes.c_int64)]


class KVSequences:
    """Sequences on a PagedKVCache, in device memory: int32 table [n, width]
    (page of each page_size positions, -1: none), lens [n] and refs [pages]
    (how many entries hold a page; 0: free)."""

    def __init__(self, table, lens, refs):
        if len(table.shape) != 2:
            raise ValueError(f"table: shape {tuple(table.shape)}")
        n, width = (int(s) for s in table.shape)
        self.table, self.lens, self.refs = table, lens, refs
        self.n, self.width, self.npages = n, width, int(refs.shape[0])
        known = {d for d in map(_device_of, (table, lens, refs)) if d is not None}
        if len(known) > 1 or min(known, default=0) < 0:
            raise ValueError(f"table, lens and refs: devices {sorted(known)} (-1: host memory), expected one device")
        self.device = known.pop() if known else None
        self.c = _SeqsC(_flat(table, "table", (n, width), _I32), _flat(lens, "lens", (n,), _I32),
                        _flat(refs, "refs", (int(refs.shape[0]),), _I32), n, width)
        self._ref = ctypes.byref(self.c)


class Rotary:
    """Rotary positions of a head's first `dims` dimensions (vs_rotary_*).

    Pair i turns by base ** (-2 i / dims) radians per position; its dimensions are
    (i, i + dims / 2) in the "half" layout, (2 i, 2 i + 1) in the "interleaved"
    one.  scaling, for contexts longer than the model's own:
      "linear"  all angles divided by factor
      "base"    base times factor ** (dims / (dims - 2))
      "ramp"    by a pair's turns within the `original` positions: up to `low` of
                them its angle is divided by factor, from `high` on it stays, in between
                a share of both; ramp_by "turns" takes the share linear in the turns,
                "index" linear in the pair's number (its ends rounded outwards)
    gain multiplies cosines and sines (None: 0.1 ln(factor) + 1 for "ramp", else 1).
    A model's "ramp" is all of these together, and the defaults are no model's: name
    low, high, ramp_by and gain as it was trained with (in use are low=1, high=4, gain=1
    over "turns", and low=1, high=32 with gain=None over "index").
    frequencies (radians per position, dims / 2 of them) stands for all that."""

    def __init__(self, head_dim: int, *, dims: int | None = None, base: float = 10000.0, layout: str = "half",
                 scaling: str = "none", factor: float = 1.0, original: int = 0, low: float = 1.0, high: float = 4.0,
                 ramp_by: str = "turns", gain: float | None = None, frequencies=None, device: int = 0):
        self._h = None
        self.head_dim, self.dims = int(head_dim), int(head_dim if dims is None else dims)
        self.device = int(device)
        if self.dims <= 0 or self.dims % 2 or self.dims > self.head_dim:
            raise ValueError(f"dims must be even and 2 to {head_dim}, got {self.dims}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be half or interleaved, got {layout}")
        if frequencies is None:
            w = self._frequencies(base, scaling, factor, original, low, high, ramp_by)
            if gain is None and scaling == "ramp":
                gain = 0.1 * math.log(factor) + 1.0
        else:
            w = np.ascontiguousarray(frequencies, np.float64)
            if w.shape != (self.dims // 2,):
                raise ValueError(f"frequencies: shape {w.shape}, expected {(self.dims // 2,)}")
        self.frequencies, self.layout, self.gain = w, layout, 1.0 if gain is None else float(gain)
        self._lib = N.load()
        h = ctypes.c_void_p()
        N.check(self._lib.vs_rotary_create(device, self.dims, w.ctypes.data_as(ctypes.c_void_p), self.gain,
                                           layout == "interleaved", ctypes.byref(h)))
        self._h = h

    def _frequencies(self, base, scaling, factor, original, low, high, ramp_by):
        dims = self.dims
        if not base > 1 or not factor > 0:
            raise ValueError(f"base must be above 1 and factor above 0, got {base} and {factor}")
        if scaling not in ("none", "linear", "base", "ramp"):
            raise ValueError(f"scaling must be none, linear, base or ramp, got {scaling}")
        if scaling == "base":
            if dims == 2:
                raise ValueError("scaling base needs more than 2 dims: a single pair turns by one radian whatever the base")
            base = base * factor ** (dims / (dims - 2))
        w = base ** (-np.arange(0, dims, 2, dtype=np.float64) / dims)
        if scaling == "linear":
            return w / factor
        if scaling != "ramp":
            return w
        if not original > 0 or not 0 < low < high:
            raise ValueError(f"ramp needs original > 0 and 0 < low < high, got {original}, {low} and {high}")
        if ramp_by == "turns":
            keep = np.clip((original * w / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        elif ramp_by == "index":
            # the pair (a real number) whose turns are `n`
            at = [dims * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (high, low)]
            first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
            keep = 1.0 - np.clip((np.arange(dims // 2) - first) / max(last - first, 1e-3), 0.0, 1.0)
        else:
            raise ValueError(f"ramp_by must be turns or index, got {ramp_by}")
        return w * keep + w / factor * (1.0 - keep)

    def close(self) -> None:
        if self._h:
            self._lib.vs_rotary_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass

    def rotate(self, x, out, positions, *, backward: bool = False, stream: int = 0) -> None:
        """out = x [rows, heads, head_dim] (f32 or bf16) turned, row i by
        positions[i] (i32) (vs_rotary_apply); out may be x.  backward: the other
        way round, a gradient of out into one of x."""
        rows, heads = int(x.shape[0]), int(x.shape[1])
        code = _code(x.dtype)
        if code < 0:
            raise ValueError(f"x: element type {x.dtype}")
        xp, xs = _rows(x, "x", (rows, heads, self.head_dim), code, self.device)
        op, os_ = _rows(out, "out", (rows, heads, self.head_dim), code, self.device)
        rc = self._lib.vs_rotary_apply(self._h, code, xp, xs[0], xs[1],
                                       _flat(positions, "positions", (rows,), _I32, self.device), rows, heads,
                                       self.head_dim, op, os_[0], os_[1], bool(backward), stream)
        if rc:
            N.check(rc)


class PagedKVCache:
    """Keys and values of every layer, in pages that stay in HBM (vs_kv_* of the C ABI)."""

    def __init__(self, npages: int, page_size: int, kv_heads: int, head_dim: int, layers: int = 1,
                 dtype: str = "bf16", device: int = 0, memory=None):
        self._h = None
        self._lib = N.load()
        self.device = int(device)
        self.npages, self.page_size, self.layers = int(npages), int(page_size), int(layers)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.code = _code(dtype)
        if self.code not in (N.VS_DTYPE_F32, N.VS_DTYPE_BF16):
            raise ValueError(f"dtype must be f32 or bf16, got {dtype}")
        self.dtype = "bf16" if self.code == N.VS_DTYPE_BF16 else "f32"
        self.memory = memory  # (kept alive)
        p = None
        if memory is not None:
            total = (self.npages * self.layers * 2 * self.kv_heads * self.page_size * self.head_dim)
            p = _flat(memory, "memory", tuple(int(s) for s in memory.shape), self.code, self.device)
            if math.prod(memory.shape) < total:
                raise ValueError(f"memory holds {math.prod(memory.shape)} values of {total}")
        h = ctypes.c_void_p()
        N.check(self._lib.vs_kv_create(device, self.npages, self.page_size, self.layers, self.kv_heads,
                                       self.head_dim, self.code, p, ctypes.byref(h)))
        self._h = h
        self._scale = 1.0 / math.sqrt(self.head_dim)

    def close(self) -> None:
        if self._h:
            self._lib.vs_kv_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass

    @property
    def page_bytes(self) -> int:
        return int(self._lib.vs_kv_page_bytes(self._h))

    def new_sequences(self, n: int, width: int, refs=None) -> KVSequences:
        """n empty sequences of up to width pages (with refs: on that cache's counts)."""
        table = DeviceArray.of(np.full((n, width), -1, np.int32), "i32", self.device)
        lens = DeviceArray.of(np.zeros(n, np.int32), "i32", self.device)
        if refs is None:
            refs = DeviceArray.of(np.zeros(self.npages, np.int32), "i32", self.device)
        return KVSequences(table, lens, refs)

    def _seqs(self, s: KVSequences):
        if s.npages != self.npages:
            raise ValueError(f"refs of {s.npages} pages on a cache of {self.npages}")
        if s.device != self.device and s.device is not None:
            raise ValueError(f"sequences on device {s.device}, a cache on device {self.device}")
        return s._ref

    def attend(self, seqs: KVSequences, q, out, *, k=None, v=None, lse=None, layer: int = 0, scale=None,
               window: int = 0, sinks: int = 0, stream: int = 0) -> None:
        """Attention of each sequence's last position (vs_kv_attend).

        q, out [n, heads, head_dim]; k, v [n, kv_heads, head_dim]: the new
        token's, stored in the same pass; lse [n, heads] f32.  window > 0: the
        last `window` positions and the first `sinks` are visible."""
        n, code, dim, dev = seqs.n, self.code, self.head_dim, self.device
        heads = int(q.shape[1])
        qp, qs = _rows(q, "q", (n, heads, dim), code, dev)
        op, os_ = _rows(out, "out", (n, heads, dim), code, dev)
        kp = vp = lp = None
        ks = vs = (0, 0)
        if k is not None or v is not None:
            if k is None or v is None:
                raise ValueError("k and v are given together or not at all")
            kp, ks = _rows(k, "k", (n, self.kv_heads, dim), code, dev)
            vp, vs = _rows(v, "v", (n, self.kv_heads, dim), code, dev)
        if lse is not None:
            lp = _flat(lse, "lse", (n, heads), N.VS_DTYPE_F32, dev)
        rc = self._lib.vs_kv_attend(
            self._h, self._seqs(seqs), layer, heads, qp, qs[0], qs[1], kp, ks[0], ks[1], vp, vs[0], vs[1],
            op, os_[0], os_[1], lp, self._scale if scale is None else scale, window, sinks, stream)
        if rc:
            N.check(rc)

    def attend_rows(self, seqs: KVSequences, q, out, *, starts=None, lse=None, layer: int = 0, scale=None,
                    causal: bool = True, window: int = 0, sinks: int = 0, stream: int = 0) -> None:
        """Attention of many rows at once (vs_kv_attend_rows): chunks of prompts,
        drafted tokens, or rows over other sequences' states.

        q, out [rows, heads, head_dim]; starts [n + 1] i32: rows starts[b] ..
        starts[b + 1] are the last positions of sequence b (none: one each), whose
        keys and values are in the cache already; lse [rows, heads] f32.  Rows
        see the positions up to their own (of them, with window > 0, the last
        `window` and the first `sinks`), or all of the sequence's if not causal."""
        rows, heads = int(q.shape[0]), int(q.shape[1])
        code, dim, dev = self.code, self.head_dim, self.device
        qp, qs = _rows(q, "q", (rows, heads, dim), code, dev)
        op, os_ = _rows(out, "out", (rows, heads, dim), code, dev)
        sp = None if starts is None else _flat(starts, "starts", (seqs.n + 1,), _I32, dev)
        lp = None if lse is None else _flat(lse, "lse", (rows, heads), N.VS_DTYPE_F32, dev)
        rc = self._lib.vs_kv_attend_rows(
            self._h, self._seqs(seqs), layer, heads, qp, qs[0], qs[1], op, os_[0], os_[1], lp, sp, rows,
            self._scale if scale is None else scale, bool(causal), window, sinks, stream)
        if rc:
            N.check(rc)

    def rows(self, seqs: KVSequences, count, starts, *, sequence=None, position=None, slot=None,
             stream: int = 0) -> None:
        """Where the rows of a batch go (vs_kv_rows): sequence b has the next
        count[b] rows (an int, or an i32 buffer [n]), for its last positions.

        starts [n + 1] i32 receives the sums of the counts; sequence, position and
        slot ([rows] i32 each, all of one length) each row's sequence, position
        and page * page_size + place on the page; -1 where there is none."""
        dev = self.device
        nrows = None
        ptrs = []
        for t, what in ((sequence, "sequence"), (position, "position"), (slot, "slot")):
            if t is None:
                ptrs.append(None)
                continue
            if nrows is None:
                nrows = int(t.shape[0])
            ptrs.append(_flat(t, what, (nrows,), _I32, dev))
        each, cp = (int(count), None) if isinstance(count, (int, np.integer)) else \
            (0, _flat(count, "count", (seqs.n,), _I32, dev))
        rc = self._lib.vs_kv_rows(self._h, self._seqs(seqs), each, cp, 2**31 - 1 if nrows is None else nrows,
                                  _flat(starts, "starts", (seqs.n + 1,), _I32, dev), *ptrs, stream)
        if rc:
            N.check(rc)

    def append(self, seqs: KVSequences, k, v, *, starts=None, layer: int = 0, rotary: Rotary | None = None, q=None,
               q_out=None, stream: int = 0) -> None:
        """Stores rows of keys and values at the sequences' last positions
        (vs_kv_append): k, v [rows, kv_heads, head_dim]; starts [n + 1] i32:
        rows starts[b] .. starts[b + 1] are sequence b's (none: one each).

        With rotary the keys are turned to their positions on the way, and the
        queries q [rows, heads, head_dim] into q_out (q itself, or another buffer)
        (vs_kv_append_rotary)."""
        rows = int(k.shape[0])
        if rotary is not None:
            return self._append_rotary(seqs, k, v, rows, starts, layer, rotary, q, q_out, stream)
        if q is not None or q_out is not None:
            raise ValueError("q and q_out go with rotary")
        kp, ks = _rows(k, "k", (rows, self.kv_heads, self.head_dim), self.code, self.device)
        vp, vs = _rows(v, "v", (rows, self.kv_heads, self.head_dim), self.code, self.device)
        sp = None if starts is None else _flat(starts, "starts", (seqs.n + 1,), _I32, self.device)
        N.check(self._lib.vs_kv_append(self._h, self._seqs(seqs), layer, kp, ks[0], ks[1], vp, vs[0], vs[1],
                                       sp, rows, stream))

    def _append_rotary(self, seqs, k, v, rows, starts, layer, rotary, q, q_out, stream) -> None:
        code, dim, dev = self.code, self.head_dim, self.device
        kp, ks = _rows(k, "k", (rows, self.kv_heads, dim), code, dev)
        vp, vs = _rows(v, "v", (rows, self.kv_heads, dim), code, dev)
        qp = op = None
        qs = os_ = (0, 0)
        heads = 0
        if q is not None or q_out is not None:
            if q is None or q_out is None:
                raise ValueError("q and q_out are given together or not at all")
            heads = int(q.shape[1])
            qp, qs = _rows(q, "q", (rows, heads, dim), code, dev)
            op, os_ = _rows(q_out, "q_out", (rows, heads, dim), code, dev)
        sp = None if starts is None else _flat(starts, "starts", (seqs.n + 1,), _I32, dev)
        rc = self._lib.vs_kv_append_rotary(
            self._h, self._seqs(seqs), layer, rotary._h, kp, ks[0], ks[1], vp, vs[0], vs[1], qp, qs[0], qs[1], heads,
            op, os_[0], os_[1], sp, rows, stream)
        if rc:
            N.check(rc)

    def read(self, seqs: KVSequences, b: int, first: int, k_out, v_out, *, layer: int = 0, stream: int = 0) -> None:
        """Positions first .. of sequence b as rows [positions, kv_heads, head_dim] (vs_kv_read)."""
        shape = (int(k_out.shape[0]), self.kv_heads, self.head_dim)
        N.check(self._lib.vs_kv_read(self._h, self._seqs(seqs), layer, b, first, shape[0],
                                     _flat(k_out, "k_out", shape, self.code, self.device),
                                     _flat(v_out, "v_out", shape, self.code, self.device), stream))

    def extend(self, seqs: KVSequences, count=1, *, stream: int = 0) -> None:
        """`count` more positions for every sequence (an int, or an i32 buffer
        [n]), with copies of shared, partly filled last pages (vs_kv_extend).
        Where it does not fit nothing changes, check() raises, and attend() and
        append() store nothing for these sequences until then."""
        if isinstance(count, (int, np.integer)):
            rc = self._lib.vs_kv_extend(self._h, self._seqs(seqs), int(count), None, stream)
        else:
            rc = self._lib.vs_kv_extend(self._h, self._seqs(seqs), 0,
                                        _flat(count, "count", (seqs.n,), _I32, self.device), stream)
        if rc:
            N.check(rc)

    def fork(self, seqs: KVSequences, parents, out: KVSequences, *, stream: int = 0) -> None:
        """out[i] = a copy of seqs[parents[i]] that shares its pages; what is
        no one's parent gives its pages back.  seqs' references go over to
        out: it is not used again but as a later fork's `out` (vs_kv_fork)."""
        rc = self._lib.vs_kv_fork(self._h, self._seqs(seqs), _list(parents, "parents", out.n, _I32, self.device),
                                  self._seqs(out), stream)
        if rc:
            N.check(rc)

    def free(self, seqs: KVSequences, ids=None, *, stream: int = 0) -> None:
        """Drops the listed sequences (an i32 buffer; None: all) (vs_kv_free)."""
        n = 0 if ids is None else int(ids.shape[0])
        if ids is not None and n == 0:
            return
        p = None if ids is None else _flat(ids, "ids", (n,), _I32, self.device)
        N.check(self._lib.vs_kv_free(self._h, self._seqs(seqs), p, n, stream))

    def evict(self, seqs: KVSequences, window: int, sinks: int = 0, *, stream: int = 0) -> None:
        """Gives back whole pages behind the window (vs_kv_evict)."""
        N.check(self._lib.vs_kv_evict(self._h, self._seqs(seqs), window, sinks, stream))

    def compact(self, seqs: KVSequences, out: KVSequences | None = None, *, others=(), moved=None, stream: int = 0) -> None:
        """Moves the pages in use to the cache's front (vs_kv_compact).

        All of them, whoever holds them: every other KVSequences on the same
        counts has to be in `others`, whose tables follow in place.  moved
        (i32 [pages]): receives where each page's contents are now, for holds
        that are in no table (vs_kv_compact_with)."""
        src, dst = self._seqs(seqs), self._seqs(seqs if out is None else out)
        if moved is None and not others:
            rc = self._lib.vs_kv_compact(self._h, src, dst, stream)
        else:
            for s in others:
                self._seqs(s)
            more = (ctypes.c_void_p * max(1, len(others)))(*(ctypes.addressof(s.c) for s in others))
            rc = self._lib.vs_kv_compact_with(self._h, src, dst, more, len(others),
                                              None if moved is None else _flat(moved, "moved", (self.npages,), _I32, self.device),
                                              stream)
        if rc:
            N.check(rc)

    def copy(self, src, dst, *, stream: int = 0) -> None:
        """Page dst[i] = page src[i] (i32 buffers) (vs_kv_copy)."""
        n = int(src.shape[0])
        N.check(self._lib.vs_kv_copy(self._h, _flat(src, "src", (n,), _I32, self.device), _flat(dst, "dst", (n,), _I32, self.device), n, stream))

    def check(self, *, stream: int = 0) -> None:
        """Waits for the stream; raises what earlier calls met on the device (vs_kv_check)."""
        N.check(self._lib.vs_kv_check(self._h, stream))


class BeamSearch:
    """The choice of the next beams and the reordering of their states (vs_beam_* of the C ABI)."""

    def __init__(self, device: int = 0):
        self._h = None
        self._lib = N.load()
        self.device = int(device)
        h = ctypes.c_void_p()
        N.check(self._lib.vs_beam_create(device, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if self._h:
            self._lib.vs_beam_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass

    def select(self, logits, scores, scores_out, tokens_out, parents_out, *, finished=None, finished_out=None,
               eos: int = -1, stream: int = 0) -> None:
        """The k best continuations of each request's beams (vs_beam_select).

        logits [requests * beams, vocab] f32 or bf16; scores [requests, beams]
        f32; finished [requests, beams] u8.  Outputs [requests, k]: scores f32,
        tokens and parents (rows of logits) i32, finished u8; in place of scores
        and finished only where k is beams."""
        dev = self.device
        try:  # (all in one: a step of one request takes as long as its Python calls)
            here = (logits.get_device() == scores.get_device() == scores_out.get_device() == tokens_out.get_device()
                    == parents_out.get_device() == dev)
        except AttributeError:
            here = False
        if not here:
            for t, what in ((logits, "logits"), (scores, "scores"), (scores_out, "scores_out"),
                            (tokens_out, "tokens_out"), (parents_out, "parents_out")):
                _on(t, what, dev)
        requests, beams = shape = scores.shape
        rows, vocab = logits.shape
        code = _SEEN.get(logits.dtype)
        if code is None:
            code = _code(logits.dtype)
        if code < 0:
            raise ValueError(f"logits: element type {logits.dtype}")
        ls = logits.stride()
        if rows != requests * beams or ls[1] != 1:
            _rows(logits, "logits", (requests * beams, vocab), code)
        _, k = out = scores_out.shape
        if out[0] != requests:
            raise ValueError(f"scores_out: shape {tuple(out)}, expected {requests} rows")
        rc = self._lib.vs_beam_select(
            self._h, logits.data_ptr(), code, ls[0] if rows > 1 else vocab, requests, beams, vocab,
            _flat(scores, "scores", shape, N.VS_DTYPE_F32),
            None if finished is None else _flat(finished, "finished", shape, _U8, dev), eos, k,
            _flat(scores_out, "scores_out", out, N.VS_DTYPE_F32), _flat(tokens_out, "tokens_out", out, _I32),
            _flat(parents_out, "parents_out", out, _I32),
            None if finished_out is None else _flat(finished_out, "finished_out", out, _U8, dev), stream)
        if rc:
            N.check(rc)

    def logprobs(self, logits, tokens, out, *, entropy=None, top_tokens=None, top_logprobs=None,
                 stream: int = 0) -> None:
        """Log probabilities of given tokens (vs_beam_logprobs).

        logits [rows, vocab] f32 or bf16; tokens [rows] i32 (-1: none, 0 comes
        out) and out [rows] f32, both or neither (None); entropy [rows] f32;
        top_tokens i32 and top_logprobs f32 [rows, k]: the k likeliest."""
        dev = self.device
        rows, vocab = logits.shape
        code = _code(logits.dtype)
        if code < 0:
            raise ValueError(f"logits: element type {logits.dtype}")
        lp, ls = _rows(logits, "logits", (rows, vocab), code, dev)
        if (tokens is None) != (out is None):
            raise ValueError("tokens and out are given together or not at all")
        if (top_tokens is None) != (top_logprobs is None):
            raise ValueError("top_tokens and top_logprobs are given together or not at all")
        f32 = N.VS_DTYPE_F32
        k = 0 if top_tokens is None else int(top_tokens.shape[1])
        rc = self._lib.vs_beam_logprobs(
            self._h, lp, code, ls[0] if rows > 1 else vocab, rows, vocab,
            None if tokens is None else _flat(tokens, "tokens", (rows,), _I32, dev),
            None if out is None else _flat(out, "out", (rows,), f32, dev),
            None if entropy is None else _flat(entropy, "entropy", (rows,), f32, dev), k,
            _flat(top_tokens, "top_tokens", (rows, k), _I32, dev) if k else None,
            _flat(top_logprobs, "top_logprobs", (rows, k), f32, dev) if k else None, stream)
        if rc:
            N.check(rc)

    def reorder(self, parents, state, out, *, tail=None, stream: int = 0) -> None:
        """Row i of `out` = row parents[i] of `state`, zeros where there is no
        such row (vs_beam_reorder).  With tail (i32, one per row) an int32
        state's last column is not copied: tail goes there."""
        code = _SEEN.get(out.dtype)
        if code is None:
            code = _code(out.dtype)
        dev = self.device
        try:
            here = state.get_device() == out.get_device() == parents.get_device() == dev
        except AttributeError:
            here = False
        if not here:
            for t, what in ((state, "state"), (out, "out"), (parents, "parents")):
                _on(t, what, dev)
        rows, cols = out.shape
        nin, wide = state.shape
        is_, os_ = state.stride(), out.stride()
        if wide != cols or _SEEN.get(state.dtype) != code or is_[1] != 1 or os_[1] != 1:
            _rows(state, "state", (nin, cols), code)
            _rows(out, "out", (rows, cols), code)
        size = _SIZES[code]
        tp, keep = None, cols
        if tail is not None:
            if code != _I32 or cols < 1:
                raise ValueError("tail needs an i32 state of at least one column")
            tp, keep = _list(tail, "tail", rows, _I32, dev), cols - 1
        pp = _list(parents, "parents", rows, _I32)
        wide = cols * size
        rc = self._lib.vs_beam_reorder(
            self._h, pp, rows, state.data_ptr(), nin, is_[0] * size if nin > 1 else wide, out.data_ptr(),
            os_[0] * size if rows > 1 else wide, keep * size, tp, stream)
        if rc:
            N.check(rc)
