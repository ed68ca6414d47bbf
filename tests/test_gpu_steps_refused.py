"""A step that attention cannot take leaves the caches as they were: their lengths, capacities and rows."""
import numpy as np
import pytest

import tract_amd as ta
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _state(caches):
    return [(c.len(), c.capacity(), c.valid_contiguous().tobytes()) for c in caches]


def _lens(caches):
    return [(c.len(), c.valid_contiguous().tobytes()) for c in caches]


def _pushed(rng, shape, dtype):
    c = ta.InPlaceKvCache(2)
    c.push(rng.standard_normal(shape, dtype=np.float32).astype(dtype))
    return c


@pytest.mark.parametrize("dtype", [F16, F32])
def test_head_sizes_that_shared_prefixes_do_not_take(rt, dtype):
    rng, d = np.random.default_rng(51), 2050
    caches = [_pushed(rng, (1, 2, n, d), dtype) for n in (3, 3, 2, 2)]
    before = _state(caches)
    q, new = (ta.DeviceTensor.from_numpy(np.ones((1, h, 1, d), dtype)) for h in (4, 2))
    for _ in range(2):
        with pytest.raises(ta.TractRocmError, match="head_dim 2050"):
            ta.inplace_kv_sdpa_eval_shared(q, new, new, *caches[:2], caches[2:3], caches[3:])
    assert _state(caches) == before


def test_more_query_rows_than_a_launch_has(rt):
    """Refused by the kernels for any head size, behind the append: nothing is counted, and the caches go on from where they were."""
    rng, d, hq, n = np.random.default_rng(52), 2, 4096, 4096
    caches = [_pushed(rng, (1, 1, m, d), F16) for m in (3, 3, 2, 2)]
    before = _lens(caches)
    q, new = ta.DeviceTensor((1, hq, n, d), F16), ta.DeviceTensor((1, 1, n, d), F16)
    with pytest.raises(ta.TractRocmError, match="too many query rows"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *caches[:2], caches[2:3], caches[3:])
    assert _lens(caches) == before
    q, new = (ta.DeviceTensor.from_numpy(np.ones((1, h, 1, d), F16)) for h in (4, 1))
    ta.inplace_kv_sdpa_eval_shared(q, new, new, *caches[:2], caches[2:3], caches[3:])
    assert [c.len() for c in caches] == [3, 3, 3, 3]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 3])
def test_head_sizes_that_steps_with_norms_do_not_take(rt, dtype, n):
    rng, d = np.random.default_rng(53), 514
    op = ta.InPlaceKvSdpa(axis=2, causal=True).state()
    op.k, op.v = (_pushed(rng, (1, 2, 2, d), dtype) for _ in range(2))
    before = _state([op.k, op.v])
    q, new = (ta.DeviceTensor.from_numpy(np.ones((1, h, n, d), dtype)) for h in (4, 2))
    cs = ta.DeviceTensor.from_numpy(np.ones((1, 1, n, d), dtype))
    dense = (2 * n * d, n * d, d, 1)
    for strides in (None, dense, (3 * n * d, n * d, d, 1)):   # (the last: values that are not dense are appended by themselves)
        with pytest.raises(ta.TractRocmError, match="head_dim 514"):
            op.eval_norm_rope_into(q, new, new, None, None, 1e-6, cs, cs, v_strides=strides)
        assert _state([op.k, op.v]) == before
    with pytest.raises(ta.TractRocmError, match="head_dim 514"):
        op.eval_into(q, new, new)
    assert _state([op.k, op.v]) == before


def test_a_scratch_over_the_inputs_of_a_step_with_norms(rt):
    """Rows of normed queries and keys would lie over what is still to be read: refused before the caches grow."""
    rng, d, n = np.random.default_rng(54), 64, 40
    kc, vc = (_pushed(rng, (1, 2, 3, d), F16) for _ in range(2))
    before = _state([kc, vc])
    q, new = (ta.DeviceTensor.from_numpy(np.ones((1, h, n, d), F16)) for h in (4, 2))
    cs, out = ta.DeviceTensor.from_numpy(np.ones((1, 1, n, d), F16)), ta.DeviceTensor((1, 4, n, d), F16)
    room = ta.DeviceTensor((8 * n * d,), F16)
    ws = ta.Workspace(1, 4, n, d)
    at = room.ptr.value
    for over in (dict(q=at + 256), dict(k=at), dict(cos=at + 512), dict(sin=at), dict(wq=at + 4 * n * d * 2)):
        a = dict(q=q.ptr, k=new.ptr, wq=None, cos=cs.ptr, sin=cs.ptr) | over
        with pytest.raises(ta.TractRocmError, match="overlap"):
            ta._lib.call("trocm_inplace_kv_sdpa_eval_norm_rope", a["q"], a["k"], new.ptr, a["wq"], None, 1e-6, a["cos"], a["sin"], 0, 1, 4, n, None, None, None,
                         kc.handle, vc.handle, out.ptr, float("nan"), 1, ws.ptr, ws.nbytes, room.ptr, room.nbytes, None)
        assert _state([kc, vc]) == before, list(over)
    ta._lib.call("trocm_inplace_kv_sdpa_eval_norm_rope", q.ptr, new.ptr, new.ptr, None, None, 1e-6, cs.ptr, cs.ptr, 0, 1, 4, n, None, None, None,
                 kc.handle, vc.handle, out.ptr, float("nan"), 1, ws.ptr, ws.nbytes, room.ptr, room.nbytes, None)
    assert kc.len() == vc.len() == 3 + n
