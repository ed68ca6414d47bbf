"""Scored attention at the ends of what its arguments may be."""
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
