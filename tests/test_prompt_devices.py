"""The prompt's calls refuse buffers that lie somewhere else than the handle's device, before anything is called."""
import pytest

from test_decode_devices import On, there  # noqa: F401


def calls(t, d):
    """Every call with all of its buffers, the i-th of them on device d(i)."""
    import vector_store as vs

    n = iter(range(99))
    at = lambda shape, dtype="bf16": On(d(next(n)), shape, dtype)  # noqa: E731
    rot = object.__new__(vs.Rotary)
    rot.__dict__.update(_h=None, _lib=t.lib, device=1, head_dim=16)
    s, c = t.seqs(1), t.cache
    return [
        lambda: c.attend_rows(s, at((9, 4, 16)), at((9, 4, 16)), starts=at((4,), "i32"), lse=at((9, 4), "f32")),
        lambda: c.rows(s, at((3,), "i32"), at((4,), "i32"), sequence=at((9,), "i32"), position=at((9,), "i32"), slot=at((9,), "i32")),
        lambda: c.append(s, at((9, 2, 16)), at((9, 2, 16)), starts=at((4,), "i32"), rotary=rot, q=at((9, 4, 16)), q_out=at((9, 4, 16))),
        lambda: rot.rotate(at((9, 4, 16)), at((9, 4, 16)), at((9,), "i32")),
        lambda: t.beams.logprobs(at((9, 50), "f32"), at((9,), "i32"), at((9,), "f32"), entropy=at((9,), "f32"),
                                 top_tokens=at((9, 3), "i32"), top_logprobs=at((9, 3), "f32")),
    ]


def test_buffers_of_the_device(there):  # noqa: F811
    for call in calls(there, lambda i: 1):
        call()
    assert there.lib.calls == 5


@pytest.mark.parametrize("where,word", [(0, "device 0"), (-1, "host memory")])
def test_a_buffer_elsewhere(there, where, word):  # noqa: F811
    sizes = (4, 5, 5, 3, 6)  # buffers of each call
    for call, size in enumerate(sizes):
        for i in range(size):
            with pytest.raises(ValueError, match=word):
                calls(there, lambda j: where if j == i else 1)[call]()
    assert there.lib.calls == 0
