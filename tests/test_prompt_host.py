"""Refusals of the prompt's entry points that need no GPU, and the plain forms' own checks."""
import ctypes

import numpy as np
import pytest

import _prompt as P

INVALID, UNSUPPORTED = 1, 4


@pytest.fixture(scope="module")
def lib():
    from vector_store import _native

    return _native.load()


def test_null_handles(lib):
    z = ctypes.c_void_p()
    assert lib.vs_kv_attend_rows(z, z, 0, 1, z, 0, 0, z, 0, 0, z, z, 0, 1.0, 1, 0, 0, z) == INVALID
    assert lib.vs_kv_rows(z, z, 0, z, 0, z, z, z, z, z) == INVALID
    assert lib.vs_kv_append_rotary(z, z, 0, z, z, 0, 0, z, 0, 0, z, 0, 0, 0, z, 0, 0, z, 0, z) == INVALID
    assert lib.vs_rotary_apply(z, 0, z, 0, 0, z, 0, 1, 2, z, 0, 0, 0, z) == INVALID
    assert lib.vs_beam_logprobs(z, z, 0, 1, 1, 1, z, z, z, 0, z, z, z) == INVALID
    assert lib.vs_rotary_create(0, 2, z, 1.0, 0, None) == INVALID
    lib.vs_rotary_destroy(z)


@pytest.mark.parametrize("dims,radians,gain,code,word", [
    (0, [1.0], 1.0, INVALID, "dims"), (3, [1.0, 1.0], 1.0, INVALID, "dims"), (-2, [1.0], 1.0, INVALID, "dims"),
    (1 << 17, None, 1.0, UNSUPPORTED, "dimensions"), (2, None, 1.0, INVALID, "radians"),
    (2, [float("nan")], 1.0, INVALID, "pair 0"), (4, [1.0, float("inf")], 1.0, INVALID, "pair 1"),
    (2, [1e300], 1.0, INVALID, "pair 0"), (2, [1.0], float("inf"), INVALID, "gain"),
])
def test_rotary_refusals(lib, dims, radians, gain, code, word):
    h = ctypes.c_void_p(5)
    w = None if radians is None else (ctypes.c_double * len(radians))(*radians)
    assert lib.vs_rotary_create(0, dims, w, gain, 0, ctypes.byref(h)) == code
    assert word in lib.vs_last_error().decode() and not h.value


@pytest.mark.parametrize("kw", [dict(dims=3), dict(dims=0), dict(dims=66), dict(layout="x"), dict(scaling="x"), dict(base=1.0),
                                dict(factor=-1.0), dict(scaling="ramp"), dict(scaling="ramp", original=9, low=3, high=3),
                                dict(scaling="ramp", original=9, ramp_by="x"), dict(frequencies=[1.0])])
def test_rotary_arguments_in_python(kw):
    import vector_store

    with pytest.raises(ValueError):
        vector_store.Rotary(64, **kw)


def test_append_takes_queries_with_rotary_only():
    from vector_store import PagedKVCache

    cache = object.__new__(PagedKVCache)  # (no GPU: the argument is looked at first)
    cache._h = None
    with pytest.raises(ValueError, match="rotary"):
        cache.append(None, np.zeros((1, 1, 16), np.float32), None, q=np.zeros(1))


def test_plain_forms_agree_with_each_other():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((5, 4, 16)), rng.standard_normal((9, 2, 16)), rng.standard_normal((9, 2, 16))
    last = np.arange(4, 9)
    out, lse, _, _ = P.attend_rows(q, k, v, P.seen_mask(last, 9, 0, 0), 0.25, "f32")
    import _decode as D

    for i, t in enumerate(last):
        o, s = D.attend(q[i], k, v, np.arange(t + 1), 0.25)
        np.testing.assert_allclose(out[i], o, rtol=1e-12)
        np.testing.assert_allclose(lse[i], s, rtol=1e-12)
    # turning there and back is the gain squared
    w = 10000.0 ** (-np.arange(8) / 8)
    for layout in ("half", "interleaved"):
        y, _ = P.turned(q, np.arange(5), w, 1.5, layout)
        back, _ = P.turned(y, np.arange(5), w, 1.5, layout, backward=True)
        np.testing.assert_allclose(back, 2.25 * q, rtol=1e-12)
        # what is seen of each other goes by the distance alone
        a, _ = P.turned(q, np.full(5, 7), w, 1.0, layout)
        b, _ = P.turned(q[::-1], np.full(5, 3), w, 1.0, layout)
        c, _ = P.turned(q, np.full(5, 104), w, 1.0, layout)
        d, _ = P.turned(q[::-1], np.full(5, 100), w, 1.0, layout)
        np.testing.assert_allclose((a * b).sum(-1), (c * d).sum(-1), rtol=1e-9, atol=1e-12)
    x = rng.standard_normal((3, 50))
    lp, ent, tt, tl = P.logprobs(x, [4, -1, 60], 50)
    p = np.exp(tl)
    np.testing.assert_allclose(p.sum(1), 1, rtol=1e-12)
    np.testing.assert_allclose(ent, -(p * tl).sum(1), rtol=1e-12)
    assert lp[0] == pytest.approx(tl[0][tt[0] == 4][0]) and lp[1] == 0 and np.isnan(lp[2])


def test_one_pair_has_no_base_to_scale():
    """Its angle is base ** 0: the factor would be ignored."""
    import vector_store

    with pytest.raises(ValueError, match="more than 2 dims"):
        vector_store.Rotary(64, dims=2, scaling="base", factor=8.0)
