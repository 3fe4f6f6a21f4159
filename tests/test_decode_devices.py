"""Buffers that lie somewhere else than the handle's device are refused before anything is called."""
import types

import pytest

from test_decode_host import Fake


class On(Fake):
    def __init__(self, device, shape, dtype="f32"):
        super().__init__(shape, dtype)
        self.where = device

    def get_device(self):
        return self.where


class Lib:
    """Answers every call with success and counts them."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0

        return call


@pytest.fixture
def there():
    """A cache and a beam search on device 1 without a library."""
    import vector_store as vs

    cache, beams = object.__new__(vs.PagedKVCache), object.__new__(vs.BeamSearch)
    lib = Lib()
    cache.__dict__.update(_h=None, _lib=lib, device=1, npages=4, page_size=32, layers=1, kv_heads=2, head_dim=16, code=1,
                          dtype="bf16", _scale=0.25)
    beams.__dict__.update(_h=None, _lib=lib, device=1)
    seqs = lambda d, n=3: vs.KVSequences(On(d, (n, 2), "i32"), On(d, (n,), "i32"), On(d, (4,), "i32"))  # noqa: E731
    return types.SimpleNamespace(cache=cache, beams=beams, lib=lib, seqs=seqs)


def calls(t, d):
    """Every call with all of its buffers, the i-th of them on device d(i)."""
    n = iter(range(99))
    at = lambda shape, dtype="bf16": On(d(next(n)), shape, dtype)  # noqa: E731
    s, o, c, b = t.seqs(1), t.seqs(1), t.cache, t.beams
    rows = lambda: at((3, 2, 16))  # noqa: E731
    return [
        lambda: c.attend(s, at((3, 4, 16)), at((3, 4, 16)), k=rows(), v=rows(), lse=at((3, 4), "f32")),
        lambda: c.append(s, rows(), rows(), starts=at((4,), "i32")),
        lambda: c.read(s, 0, 0, rows(), rows()),
        lambda: c.extend(s, at((3,), "i32")),
        lambda: c.fork(s, at((3,), "i32"), o),
        lambda: c.free(s, at((2,), "i32")),
        lambda: c.compact(s, moved=at((4,), "i32")),
        lambda: c.copy(at((2,), "i32"), at((2,), "i32")),
        lambda: b.select(at((6, 50), "f32"), at((2, 3), "f32"), at((2, 4), "f32"), at((2, 4), "i32"), at((2, 4), "i32"),
                         finished=at((2, 3), "u8"), finished_out=at((2, 4), "u8")),
        lambda: b.reorder(at((6,), "i32"), at((6, 8), "i32"), at((6, 8), "i32"), tail=at((6,), "i32")),
    ]


def test_buffers_on_the_handles_device_are_taken(there):
    every = calls(there, lambda i: 1)
    for f in every:
        f()
    assert there.lib.calls == len(every)


@pytest.mark.parametrize("where", [-1, 0])
@pytest.mark.parametrize("place", range(7))
def test_a_buffer_elsewhere_is_refused(there, where, place):
    for at in range(len(calls(there, None))):
        seen = []

        def device(i):
            seen.append(i)
            return where if i == place else 1

        f = calls(there, device)[at]
        if place == 0:
            with pytest.raises(ValueError, match="host memory" if where < 0 else "device 0"):
                f()
        else:
            try:
                f()
            except ValueError as e:
                assert place in seen and ("host memory" if where < 0 else "device 0") in str(e)
            else:
                assert place not in seen  # (it has fewer buffers)
                there.lib.calls -= 1
    assert there.lib.calls == 0


def test_sequences_elsewhere_are_refused(there):
    import vector_store as vs

    for d in (-1, 0):
        with pytest.raises(ValueError, match="device"):
            there.cache.attend(there.seqs(d), On(1, (3, 4, 16), "bf16"), On(1, (3, 4, 16), "bf16"))
    with pytest.raises(ValueError, match="device"):
        there.cache.compact(there.seqs(1), there.seqs(0))
    with pytest.raises(ValueError, match="one device"):
        vs.KVSequences(On(1, (3, 2), "i32"), On(1, (3,), "i32"), On(0, (4,), "i32"))
    with pytest.raises(ValueError, match="one device"):
        vs.KVSequences(On(1, (3, 2), "i32"), On(-1, (3,), "i32"), On(1, (4,), "i32"))
    assert there.lib.calls == 0


def test_buffers_that_do_not_say_are_trusted(there):
    s = there.seqs(1)
    there.cache.attend(s, Fake((3, 4, 16), "bf16"), Fake((3, 4, 16), "bf16"))
    assert there.lib.calls == 1


@pytest.mark.parametrize("count", [3, "int32", "int64", "uint8"])
def test_counts_of_any_whole_type(there, count):
    """numpy's whole numbers are numbers, not buffers."""
    import numpy as np

    there.cache.extend(there.seqs(1), count if isinstance(count, int) else getattr(np, count)(3))
    assert there.lib.calls == 1
