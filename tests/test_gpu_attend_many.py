"""Attention over many sequences at a time: the division of their work, and that it grows with them."""
import time

import numpy as np
import pytest

import _decode as D
from test_gpu_attend import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [384, 385, 1024, 1025, 2500])
def test_many_sequences_in_wide_tables(vs, dtype, n):
    """Empty, short and a few long ones, in tables so wide that they may be split; windows too."""
    lens = [(i * 37) % 90 if i % 7 else 0 for i in range(n)]
    lens[n // 3], lens[n - 1], lens[5] = 1280, 1100, 700
    c = Case(vs, lens, 2, 1, 16, 32, dtype, width=40)
    c.compare(c.run())
    c.compare(c.run(window=300, sinks=33), 300, 33)


@pytest.mark.parametrize("n", [500, 1500])
def test_many_equal_and_many_empty(vs, n):
    for lens in ([40] * n, [0] * n, [0] * (n - 1) + [1280]):
        c = Case(vs, lens, 2, 1, 16, 32, "bf16", width=40)
        c.compare(c.run())


def test_time_grows_with_the_sequences(vs):
    """Eight times the sequences take less than 16 times as long (a division of the work that reads all lengths
    in every workgroup took 29 times as long)."""
    A = vs.DeviceArray
    pages, dim, width = 4096, 128, 40
    cache = vs.PagedKVCache(pages, 32, 8, dim)
    rng = np.random.default_rng(0)

    def seconds(n):
        table, lens = rng.integers(0, pages, (n, width)), rng.integers(32, 1200, n)  # (pages read by many)
        seqs = vs.KVSequences(A.of(table, "i32"), A.of(lens, "i32"), A.of(np.zeros(pages), "i32"))
        q, out = A.of(np.zeros((n, 8, dim)), "bf16"), A((n, 8, dim), "bf16")
        took = []
        for _ in range(5):
            cache.check()
            t0 = time.perf_counter()
            for _ in range(4):
                cache.attend(seqs, q, out)
            cache.check()
            took.append(time.perf_counter() - t0)
        return min(took)

    few, many = seconds(2048), seconds(16384)
    assert many < 16 * few, (few, many)
    cache.close()


def test_recorded_and_on_one_handle_with_few(vs):
    """A plan of many sequences and calls of few use the scratch in turn."""
    lens = [(i * 53) % 120 for i in range(700)]
    c = Case(vs, lens, 2, 1, 16, 32, "bf16", width=40)
    few = vs.KVSequences(c.vs.DeviceArray.of(c.table[:9], "i32"), c.vs.DeviceArray.of(c.lens[:9], "i32"), c.seqs.refs)
    A = vs.DeviceArray
    q9, out9 = A.of(c.qb[:9], "bf16"), A((9, 2, 16), "bf16")
    first = c.run()
    c.compare(first)
    for _ in range(3):
        c.cache.attend(few, q9, out9)
        again = c.run()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    got = D.from_bf16(out9.numpy())
    for b in range(9):
        args = (c.q[b], c.k[b], c.v[b], np.arange(lens[b]), 0.25)
        D.assert_rounded(got[b], D.attend(*args)[0], D.attend_tolerance(*args, "bf16")[0], "bf16")
