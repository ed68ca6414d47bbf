"""Recorded calls are replayed after their operators took larger shapes: the workspace that a graph knows stays, and the results too."""
import ctypes as C

import numpy as np
import pytest

import tract_amd as ta
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16 = np.float16


def _device(rng, *shape, scale=1.0):
    return ta.DeviceTensor.from_numpy((rng.standard_normal(shape, dtype=np.float32) * scale).astype(F16))


def _scrub(t):
    a = np.full(t.shape, np.nan, t.dtype)
    ta._lib.call("trocm_h2d", t.ptr, a.ctypes.data_as(C.c_void_p), t.nbytes, None)
    ta.synchronize()


@pytest.mark.parametrize("kind", ["shared", "scored"])
def test_replayed_after_a_larger_call(rt, kind):
    hip = C.CDLL("libamdhip64.so")

    def ok(rc):
        assert rc == 0, f"HIP error {rc}"

    rng, stream = np.random.default_rng(71), ta.Stream()
    hq, hkv, d = 8, 2, 128

    def calls(op, n):
        """The call of n sequences, and its output: each in several parts."""
        out = ta.DeviceTensor((n, hq, 1, d), F16)
        q, k, v = _device(rng, n, hq, 1, d, scale=2.0), _device(rng, n, hkv, 900, d), _device(rng, n, hkv, 900, d)
        if kind == "shared":
            pk, pv = _device(rng, 1, hkv, 3000, d), _device(rng, 1, hkv, 3000, d)
            return lambda: op.eval(q, pk, pv, k, v, [900] * n, stream=stream, out=out), out
        return lambda: op.eval(q, k, v, stream=stream, out=out), out

    op = ta.SharedPrefixSdpa() if kind == "shared" else ta.ScoredSdpa(softcap=20.0)
    small, out = calls(op, 2)
    small()
    want = out.to_numpy(stream).tobytes()
    handle = stream.handle if isinstance(stream.handle, C.c_void_p) else C.c_void_p(stream.handle)
    graph, run = C.c_void_p(), C.c_void_p()
    ok(hip.hipStreamBeginCapture(handle, C.c_int(1)))
    small()
    ok(hip.hipStreamEndCapture(handle, C.byref(graph)))
    ok(hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
    for n in (1, 60, 200):
        larger, larger_out = calls(op, n)
        fresh, fresh_out = calls(ta.SharedPrefixSdpa() if kind == "shared" else ta.ScoredSdpa(softcap=20.0), n)
        for _ in range(2):
            larger(), fresh()
            _scrub(out)
            ok(hip.hipGraphLaunch(run, handle))
            stream.synchronize()
            assert out.to_numpy(stream).tobytes() == want, n
            assert np.isfinite(larger_out.to_numpy(stream)).all() and np.isfinite(fresh_out.to_numpy(stream)).all()
        _scrub(out)
        small()
        assert out.to_numpy(stream).tobytes() == want, n
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
