"""Scored attention and shared prefixes where scores are so far apart that the largest one is all there is, and prefix lengths of any value."""
import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, scored
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(1, 32, 8, 1000, 1000, 128), (2, 4, 2, 1, 3000, 64), (1, 4, 2, 30, 200, 64), (1, 2, 1, 5, 40, 48)], ids=str)
def test_prefix_lengths_of_any_value(rt, dtype, shape):
    """Negative ones are no prefix, those past the last key all of it."""
    b, hq, hkv, n, t, d = shape
    if dtype == F32 and n == 1000:
        shape = b, hq, hkv, n, t, d = 1, 4, 2, 300, 300, 128
    rng = np.random.default_rng(61)
    q, k, v = _rows(rng, (b, hq, n, d), dtype, 2.0), _rows(rng, (b, hkv, t, d), dtype), _rows(rng, (b, hkv, t, d), dtype)
    none, whole = scored(q, k, v), scored(q, k, v, causal=False)
    for length, want in ((-(2**31), none), (-(2**31) + 1, none), (-1, none), (0, none), (t, whole), (2**31 - 1, whole)):
        got = ta.ScoredSdpa().eval(q, k, v, prefix_lens=np.full(b, length, np.int32)).to_numpy()
        assert_within(got, *want, what=f"a prefix of {length}")


SHAPES = [(1, 32, 8, 1000, 1000, 128), (1, 64, 8, 1000, 1000, 64), (1, 8, 2, 1, 3000, 128), (1, 8, 2, 40, 400, 64)]


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("slope,scale", [(1e5, None), (1e6, None), (3e7, None), (1e30, None), (1e30, 2e-6), (1e12, 2e-6)])
def test_slopes_that_leave_one_key(rt, shape, cap, slope, scale):
    """A step in distance is at least 1e5 and far more than a step of 32 bits at the largest distance: a row is its own key's values,
    or, where scores rise with the distance, the first key's."""
    b, hq, hkv, n, t, d = shape
    rng = np.random.default_rng(62)
    q, k, v = _rows(rng, (b, hq, n, d), F16), _rows(rng, (b, hkv, t, d), F16), _rows(rng, (b, hkv, t, d), F16)
    slopes = (slope * rng.uniform(1.0, 2.0, hq) * np.where(np.arange(hq) % 2, -1.0, 1.0)).astype(F32).clip(-1e30, 1e30)
    got = ta.ScoredSdpa(scale, cap).eval(q, k, v, slopes=slopes).to_numpy()
    each = np.repeat(v, hq // hkv, axis=1)
    want = np.where((slopes > 0)[None, :, None, None], each[:, :, t - n :], each[:, :, :1])
    assert np.array_equal(got, want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["prompt", "token", "prefix"])
def test_products_that_leave_one_key(rt, kind, d):
    """Scores of 7e8 and more, a score's step of 32 bits and its reference's far over 1, two keys alike above all others."""
    rng = np.random.default_rng(63)
    hq, hkv, t = 32, 4, 5000 if kind == "prefix" else 2000
    n = t if kind == "prompt" else 1
    seqs = 40 if kind == "prefix" else 1
    size = rng.integers(1, 900, (hkv, t)).astype(np.float32)
    first, second = 150 + 7 * np.arange(hkv), 1900 - 11 * np.arange(hkv)
    for g in range(hkv):
        size[g, [first[g], second[g]]] = 1000.0
    sign = rng.choice([-1.0, 1.0], d).astype(np.float32)
    k = (32.0 * size[None, :, :, None] * sign).astype(F16)
    v = _rows(rng, (1, hkv, t, d), F16)
    q = (rng.integers(3000, 60000, (seqs, hq, n, 1)).astype(np.float32) * sign).astype(F16)
    if kind == "prefix":
        none = np.zeros((seqs, hkv, 1, d), F16)
        got = ta.SharedPrefixSdpa().eval(q, k, v, none, none, [0] * seqs).to_numpy()
    else:
        got = ta.ScoredSdpa(is_causal=False).eval(q, k, v).to_numpy()
    for h in range(hq):
        g = h * hkv // hq
        want = (v[0, g, first[g]].astype(np.float64) + v[0, g, second[g]]) / 2
        assert np.allclose(got[:, h].astype(np.float64), want, rtol=2.0**-11, atol=2.0**-24), (h, got[0, h, 0], want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["prompt", "token", "prefix"])
def test_products_a_step_of_32_bits_apart(rt, kind, d):
    """Scores of about 1e8 to 3e10 that differ by a few steps of 32 bits, each of which is a factor that no weight has: whichever keys they
    leave, a row is inside what the values span."""
    rng = np.random.default_rng(64)
    hq, hkv, t = 32, 4, 5000 if kind == "prefix" else 2000
    n = t if kind == "prompt" else 1
    seqs = 40 if kind == "prefix" else 1
    k = np.full((1, hkv, t, d), 32000.0, F16)
    k[..., -1] = rng.integers(0, 400, (1, hkv, t)) / 4
    v = rng.uniform(1.0, 2.0, (1, hkv, t, d)).astype(F16)
    q = np.repeat(2.0 ** rng.uniform(8.0, 15.9, (seqs, hq, n, 1)), d, axis=-1).astype(F16)
    if kind == "prefix":
        none = np.zeros((seqs, hkv, 1, d), F16)
        got = ta.SharedPrefixSdpa().eval(q, k, v, none, none, [0] * seqs).to_numpy()
    else:
        got = ta.ScoredSdpa(is_causal=False).eval(q, k, v).to_numpy()
    assert np.isfinite(got).all() and got.min() >= 1.0 - 2.0**-11 and got.max() <= 2.0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cap,scale", [(1e-30, 1e9), (1e-30, -1e30), (1e-6, 1e34), (2.0, 3e38)])
@pytest.mark.parametrize("shape", [(1, 32, 8, 1000, 1000, 128), (1, 8, 2, 1, 900, 64), (1, 2, 1, 5, 40, 48)], ids=str)
def test_scales_far_above_the_cap(rt, dtype, cap, scale, shape):
    """A scale that f32 cannot hold once divided by the cap: a product of zero is still a score of zero, any other the cap or its opposite."""
    b, hq, hkv, n, t, d = shape
    if dtype == F32 and n == 1000:
        b, hq, hkv, n, t, d = 1, 4, 2, 300, 300, 128
    rng = np.random.default_rng(65)
    q = np.zeros((b, hq, n, d), dtype)
    q[:, ::2, :, 0] = 1.0
    k = _rows(rng, (b, hkv, t, d), dtype)
    k[..., 0] = rng.choice([-2.0, 2.0], (b, hkv, t))
    v = _rows(rng, (b, hkv, t, d), dtype)
    got = ta.ScoredSdpa(scale, cap).eval(q, k, v).to_numpy()
    signs = np.sign(scale) * np.sign(k)
    want = scored(q, signs.astype(dtype), v, scale=cap)    # the score: cap times the product's sign
    assert_within(got, want[0], want[1] + 1e-6 * np.abs(v).max())
