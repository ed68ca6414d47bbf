"""Steps over a shared prefix whose rows are not whole 4-byte words, or lie where no 4-byte access fits."""
import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, shared
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


@pytest.mark.parametrize("dtype,d", [(F16, 7), (F16, 1), (F16, 33), (F32, 7), (F16, 6)])
@pytest.mark.parametrize("n_seq,hq,hkv,shift", [(3, 6, 3, 0), (90, 2, 2, 0), (2, 4, 2, 1)])   # 90: more than the arguments of one launch hold
def test_steps(rt, dtype, d, n_seq, hq, hkv, shift):
    rng = np.random.default_rng(31)
    prefix = [ta.InPlaceKvCache(2) for _ in range(2)]
    pk, pv = (_rows(rng, (1, hkv, 5, d), dtype) for _ in range(2))
    prefix[0].push(pk), prefix[1].push(pv)
    ks, vs = ([ta.InPlaceKvCache(2) for _ in range(n_seq)] for _ in range(2))
    own_k, own_v = ([np.zeros((hkv, 0, d), dtype) for _ in range(n_seq)] for _ in range(2))
    for sq in (1, 2, 3, 1):
        q = _rows(rng, (n_seq, hq, sq, d), dtype, 2.0)
        new = [_rows(rng, (n_seq, hkv, sq, d), dtype) for _ in range(2)]
        flat = [ta.DeviceTensor.from_numpy(np.concatenate([np.zeros(shift, dtype), t.reshape(-1)])) for t in new]
        dk, dv = (ta.DeviceTensor(t.shape, dtype, ptr=f.ptr.value + shift * t.itemsize, owner=f) for t, f in zip(new, flat))
        got = ta.inplace_kv_sdpa_eval_shared(ta.DeviceTensor.from_numpy(q), dk, dv, *prefix, ks, vs).to_numpy()
        own_k, own_v = ([np.concatenate([o, t], axis=1) for o, t in zip(own, n)] for own, n in zip((own_k, own_v), new))
        for c, o in zip(ks + vs, own_k + own_v):
            assert c.valid_contiguous().tobytes() == o[None].tobytes()
        assert_within(got, *shared(q, pk[0], pv[0], own_k, own_v))
