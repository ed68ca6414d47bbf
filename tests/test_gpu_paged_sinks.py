"""Attention over pages beside a key that has nearly all of the weight and a value of next to nothing: the result is what the others leave."""
import numpy as np
import pytest

import tract_amd as ta
from tests import paged_ref as ref
from tests.attention_ref import assert_within
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy


def _attend(q, k, v, lens, page):
    """k, v [n_seq, kv_heads, tokens, head_dim] of sequences one behind the other in the pool."""
    n, hkv, t, d = k.shape
    pages = t // page
    pool = lambda x: np.ascontiguousarray(x.reshape(n, hkv, pages, page, d).transpose(0, 2, 1, 3, 4)).reshape(n * pages, hkv, page, d)  # noqa: E731
    table, lens = np.arange(n * pages, dtype=I32).reshape(n, pages), np.asarray(lens, I32)
    want, bound = ref.attend(q, pool(k), pool(v), table, lens, scale=1.0)
    got = ta.PagedSdpa(1.0).eval(up(q), up(pool(k)), up(pool(v)), up(table), up(lens)).to_numpy()
    assert_within(got, want, bound, f"{lens.tolist()} {q.shape}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("below", [9.3, 14.7, 17.4, 20.6, 22.6, 25.5, 28.3])
@pytest.mark.parametrize("d,hq,sq", [(64, 4, 1), (128, 4, 1), (64, 8, 5), (128, 8, 3), (96, 2, 1)])
def test_a_key_with_nearly_all_of_the_weight(rt, dtype, below, d, hq, sq):
    """The others' scores `below` halvings under its own, all the same (weights are rounded the same way), nearly so, or rising from key to key."""
    rng, hkv, page, t = np.random.default_rng(d + hq), 2, 16, 1600
    q = np.full((3, hq, sq, d), 1 / 8, dtype)
    v = (0.5 + rng.random((3, hkv, t, d))).astype(dtype)
    k = np.zeros((3, hkv, t, d), dtype)
    k[1] = (rng.standard_normal((hkv, t, d)) / 16).astype(dtype)
    k[2] = (np.arange(t)[None, :, None] / t * 8 / d).astype(dtype)
    at = [0, 777, 1300]
    for i in range(3):
        k[i, :, at[i]] = below * np.log(2) * 8 / d
        v[i, :, at[i]] = 0
    _attend(q, k, v, [1600, 1599, 1411], page)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_scores_far_from_zero(rt, dtype):
    """References whose last place is a sixteenth, or 2 and more: no weight is past the type's largest."""
    rng, page, t, d = np.random.default_rng(2), 16, 400, 64
    for size in (1e5, 3e7, 1.2e8, 1e9):
        q = np.full((4, 2, 2, d), 64, dtype)
        k = np.full((4, 1, t, d), size / d / 64 if dtype == F32 or size < 2e8 else 45000.0, dtype)
        k[1:3] *= -1
        k[2:, :, 100:200] *= dtype(0.75)
        k[:, :, 37] *= dtype(1.25)
        _attend(q, k, (0.5 + rng.random((4, 1, t, d))).astype(dtype), [400, 400, 399, 200], page)
