"""Host side of the operators around attention: what Python passes on and refuses, with the library's calls recorded (no device)."""
import types

import numpy as np
import pytest

from tract_amd import TractRocmError, scored
from tract_amd.runtime import DeviceTensor

F16 = np.dtype(np.float16)
AT = 1 << 20   # an address that nothing reads


def _tensor(*shape, dtype=F16):
    return DeviceTensor(shape, dtype, ptr=AT)


def _cache(shape):
    return types.SimpleNamespace(_h=1, handle=1, _shape=shape)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(scored, "call", lambda name, *args: made.append(name))
    return made


@pytest.mark.parametrize("d", [64, 256])
def test_a_shared_step_refuses_queries_of_another_head_size_than_the_caches(calls, d):
    """The library sizes q, the new rows and the output by the caches' head size: smaller tensors would be read and written past their ends."""
    caches = [_cache((1, 2, 0, 128)) for _ in range(4)]
    prefix = [_cache((1, 2, 9, 128)) for _ in range(2)]
    q, new = _tensor(2, 4, 1, d), _tensor(2, 2, 1, d)
    ws = types.SimpleNamespace(ptr=AT, nbytes=0)
    for rows in (new, None):
        with pytest.raises(TractRocmError, match="head size"):
            scored.inplace_kv_sdpa_eval_shared(q, rows, rows, *prefix, caches[:2], caches[2:], workspace=ws, out=_tensor(2, 4, 1, d))
    with pytest.raises(TractRocmError, match="rank 4"):
        scored.inplace_kv_sdpa_eval_shared(_tensor(2, 1, 128), None, None, *prefix, caches[:2], caches[2:], workspace=ws)
    assert not calls
    q, new = _tensor(2, 4, 1, 128), _tensor(2, 2, 1, 128)
    scored.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, caches[:2], caches[2:], workspace=ws, out=_tensor(2, 4, 1, 128))
    assert calls == ["trocm_inplace_kv_sdpa_eval_shared"]
