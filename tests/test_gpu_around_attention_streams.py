"""The operators around attention on several streams, from several threads, and recorded into graphs: always the plain call's bytes."""
import ctypes as C
import threading

import numpy as np
import pytest

import tract_amd as ta
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32


def _device(rng, shape, dtype=F16, scale=1.0):
    return ta.DeviceTensor.from_numpy((rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype))


def _calls(seed, dtype=F16):
    """name -> (call(stream), outputs): each with outputs and, where one is taken, an operator and a workspace of its own."""
    rng = np.random.default_rng(seed)
    calls = {}
    # single tokens over long keys, joined inside the kernel; a prompt; a prompt in documents
    for name, (b, hq, hkv, n, t, d), rules in (("tokens", (3, 8, 2, 1, 3000, 128), {}), ("prompt", (1, 8, 2, 700, 700, 64), {}), ("full", (1, 32, 8, 1000, 1000, 128), {}),
                                               ("documents", (2, 14, 2, 300, 340, 64), {"documents": np.repeat(np.arange(10, dtype=I32), 34)[None].repeat(2, axis=0)})):
        q, k, v, out = _device(rng, (b, hq, n, d), dtype, 3.0), _device(rng, (b, hkv, t, d), dtype), _device(rng, (b, hkv, t, d), dtype), ta.DeviceTensor((b, hq, n, d), dtype)
        rules = {x: ta.DeviceTensor.from_numpy(y) for x, y in rules.items()}
        op = ta.ScoredSdpa(softcap=20.0)
        calls[name] = (lambda stream, op=op, q=q, k=k, v=v, out=out, rules=rules: op.eval(q, k, v, stream=stream, out=out, **rules)), [out]
    # sequences behind a prefix: few (joined inside the kernel), and many (tall tiles, joined by a launch of their own)
    for name, n, p, longest in (("few", 5, 900, 70), ("many", 70, 1500, 90)):
        hq, hkv, d = 8, 2, 128
        q, pk, pv, out = _device(rng, (n, hq, 1, d), dtype, 2.0), _device(rng, (1, hkv, p, d), dtype), _device(rng, (1, hkv, p, d), dtype), ta.DeviceTensor((n, hq, 1, d), dtype)
        k, v, lens = _device(rng, (n, hkv, longest, d), dtype), _device(rng, (n, hkv, longest, d), dtype), [int(x) for x in rng.integers(0, longest, n)]
        op = ta.SharedPrefixSdpa()
        calls[name] = (lambda stream, op=op, a=(q, pk, pv, k, v, lens), out=out: op.eval(*a, stream=stream, out=out)), [out]
    q, k, w, cs = _device(rng, (2, 8, 33, 128), dtype), _device(rng, (2, 2, 33, 128), dtype), _device(rng, (128,), dtype), _device(rng, (1, 1, 33, 128), dtype)
    qo, ko, op = ta.DeviceTensor(q.shape, dtype), ta.DeviceTensor(k.shape, dtype), ta.QkNormRope(1e-6)
    calls["norm"] = (lambda stream: op.eval(q, k, w, w, cs, cs, stream=stream, q_out=qo, k_out=ko)), [qo, ko]
    return calls


def _bytes(outs, stream=None):
    return [o.to_numpy(stream).tobytes() for o in outs]


def _scrub(outs):
    for o in outs:
        a = np.full(o.shape, np.nan, o.dtype)
        ta._lib.call("trocm_h2d", o.ptr, a.ctypes.data_as(C.c_void_p), o.nbytes, None)
    ta.synchronize()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_two_streams_at_once(rt, dtype):
    a, b = _calls(1, dtype), _calls(1, dtype)
    want = {}
    for name, (call, outs) in a.items():
        call(None)
        want[name] = _bytes(outs)
    streams = ta.Stream(), ta.Stream()
    for _ in range(5):
        for calls, stream in zip((a, b), streams):
            for call, _ in calls.values():
                call(stream)
    for calls, stream in zip((a, b), streams):
        for name, (_, outs) in calls.items():
            assert _bytes(outs, stream) == want[name], name


def test_threads_with_streams_of_their_own(rt):
    want = {}
    for name, (call, outs) in _calls(2).items():
        call(None)
        want[name] = _bytes(outs)
    ta.synchronize()
    wrong = []

    def work():
        try:
            calls, stream = _calls(2), ta.Stream()
            for _ in range(10):
                for call, _ in calls.values():
                    call(stream)
            wrong.extend(name for name, (_, outs) in calls.items() if _bytes(outs, stream) != want[name])
        except Exception as e:   # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_captured_and_replayed_with_a_shared_workspace(rt):
    """Two graphs of the same calls, replayed in turn between eager calls of the same operators (one stream, one workspace each)."""
    hip = C.CDLL("libamdhip64.so")

    def ok(rc):
        assert rc == 0, f"HIP error {rc}"

    calls, stream = _calls(3), ta.Stream()
    want = {}
    for name, (call, outs) in calls.items():
        call(stream)
        want[name] = _bytes(outs, stream)
    handle = stream.handle if isinstance(stream.handle, C.c_void_p) else C.c_void_p(stream.handle)
    graphs = []
    for _ in range(2):
        graph, run = C.c_void_p(), C.c_void_p()
        ok(hip.hipStreamBeginCapture(handle, C.c_int(1)))
        for call, _ in calls.values():
            call(stream)
        ok(hip.hipStreamEndCapture(handle, C.byref(graph)))
        ok(hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
        graphs.append((graph, run))
    for turn in range(6):
        for _, (_, outs) in calls.items():
            _scrub(outs)
        ok(hip.hipGraphLaunch(graphs[turn % 2][1], handle))
        stream.synchronize()
        for name, (_, outs) in calls.items():
            assert _bytes(outs, stream) == want[name], f"replay {turn}: {name}"
        for name, (call, outs) in calls.items():
            _scrub(outs)
            call(stream)
            assert _bytes(outs, stream) == want[name], f"eager call after replay {turn}: {name}"
    for graph, run in graphs:
        ok(hip.hipGraphExecDestroy(run))
        ok(hip.hipGraphDestroy(graph))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_workspace_for_operators_in_turn(rt, dtype):
    """The dense, the shared and the scored attention leave a workspace ready for each other."""
    rng = np.random.default_rng(4)
    b, hq, hkv, t, d = 6, 8, 2, 2500, 128
    q, k, v, out = _device(rng, (b, hq, 1, d), dtype, 2.0), _device(rng, (b, hkv, t, d), dtype), _device(rng, (b, hkv, t, d), dtype), ta.DeviceTensor((b, hq, 1, d), dtype)
    ws = ta.Workspace(b, hq, 1, d, nbytes=max(ta.Workspace.bytes_for(b, hq, 1, d), ta.Workspace.shared_bytes_for(b, hq, 1, d)))
    code, nan, lens = 0 if dtype == F32 else 1, float("nan"), (C.c_int64 * b)(*range(5, 5 + b))
    st = (C.c_int64 * 3)(hkv * t * d, t * d, d)
    steps = {
        "scored": lambda: ta._lib.call("trocm_sdpa_scored", q.ptr, k.ptr, v.ptr, out.ptr, code, b, hq, hkv, 1, t, d, None, nan, 30.0, None, None, None, 1, ws.ptr, ws.nbytes, None),
        "shared": lambda: ta._lib.call("trocm_sdpa_shared_prefix", q.ptr, code, b, hq, hkv, 1, d, k.ptr, v.ptr, t, (C.c_int64 * 2)(t * d, d), k.ptr, v.ptr, st, lens, out.ptr, nan, 1,
                                       ws.ptr, ws.nbytes, None),
        "dense": lambda: ta._lib.call("trocm_sdpa", q.ptr, k.ptr, v.ptr, None, out.ptr, code, b, hq, hkv, 1, t, d, None, 0, 0, nan, 1, ws.ptr, ws.nbytes, None),
    }
    want = {}
    for name, step in steps.items():
        step()
        want[name] = _bytes([out])
    for name in ("dense", "scored", "dense", "shared", "scored", "shared", "dense", "dense", "shared", "shared", "scored", "scored") * 2:
        _scrub([out])
        steps[name]()
        assert _bytes([out]) == want[name], name
