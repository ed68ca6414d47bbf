"""The operators over pages together, as serving and beam search use them; on several streams and threads; recorded and replayed."""
import ctypes as C
import threading

import numpy as np
import pytest

import tract_amd as ta
from tests import attention_ref
from tests import paged_ref as ref
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy


class Plain:
    """Sequences as lists of rows: what PagedKvCache stands for."""

    def __init__(self, seqs, layers):
        self.rows = [[[] for _ in range(2 * layers)] for _ in range(seqs)]

    def append(self, layer, i, k, v):
        self.rows[i][2 * layer].append(k)
        self.rows[i][2 * layer + 1].append(v)

    def reorder(self, parents):
        self.rows = [[list(t) for t in self.rows[p]] if p >= 0 else [[] for _ in self.rows[0]] for p in parents]

    def check(self, layer, q, got, what):
        for i, row in enumerate(self.rows):
            n, (hq, sq, d) = len(row[2 * layer]), q[i].shape
            if n == 0:
                assert (got[i] == 0).all(), what
                continue
            k, v = (np.stack(row[2 * layer + x], axis=1) for x in range(2))
            sees = np.arange(n)[None, :] <= n - sq + np.arange(sq)[:, None]
            for h in range(hq):
                kv = h * k.shape[0] // hq
                want, bound = attention_ref.attend(q[i, h], k[kv], v[kv], q.dtype, sees=sees)
                attention_ref.assert_within(got[i, h], want, bound, f"{what}, sequence {i}, head {h}")


def _held(cache):
    """Every page is held as often as refs says, or free once."""
    table, lens = cache.table.to_numpy(), cache.lens()
    refs, free = cache._now("refs").to_numpy(), cache._now("free").to_numpy()[: cache.free()]
    held = np.concatenate([row[: -(-int(n) // cache.page_size)] for row, n in zip(table, lens)])
    np.testing.assert_array_equal(np.bincount(held, minlength=cache.n_pages), refs)
    assert sorted(free) == list(np.flatnonzero(refs == 0))


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(F16, 4, 2, 64, 16), (F32, 4, 4, 64, 16), (F16, 8, 2, 128, 32), (F16, 2, 1, 40, 5)])
def test_beam_search_over_pages(rt, dtype, hq, hkv, d, page):
    """Prompts for the first beam of every request, shared by the others; then steps that choose continuations and go on from their beams."""
    rng, batch, beams, layers, vocab, eos = np.random.default_rng(page), 3, 4, 2, 1000, 7
    n = batch * beams
    cache, plain = ta.PagedKvCache(200, page, hkv, d, n, 200, dtype, layers=layers), Plain(n, layers)
    select = ta.BeamSelect(beams, eos=eos)

    def step(new, sq):
        """new [n] tokens a sequence; attends with the last sq."""
        tokens = int(new.sum())
        cache.plan(up(new.astype(I32)), tokens)
        starts = np.concatenate([[0], np.cumsum(new)])
        for layer in range(layers):
            k, v = (rng.standard_normal((tokens, hkv, d)).astype(dtype) for _ in range(2))
            cache.append(layer, up(k), up(v))
            for i in range(n):
                for t in range(starts[i], starts[i + 1]):
                    plain.append(layer, i, k[t], v[t])
        assert cache.refused() == 0
        np.testing.assert_array_equal(cache.lens(), [len(r[0]) for r in plain.rows])
        for layer in range(layers):
            q = (rng.standard_normal((n, hq, sq, d)) * 2).astype(dtype)
            plain.check(layer, q, cache.attend(layer, up(q)).to_numpy(), f"layer {layer}")

    prompt = np.zeros(n, int)
    prompt[::beams] = rng.integers(1, 3 * page + 2, batch)
    step(prompt, 1)
    first = np.repeat(np.arange(0, n, beams), beams)
    cache.reorder(up(first.astype(I32)))
    plain.reorder(first)
    _held(cache)
    scores, ended = np.zeros((batch, beams), F32), np.zeros((batch, beams), I32)
    scores[:, 1:] = -np.inf      # (all beams are alike: continuations of the first alone)
    for turn in range(2 * page + 3):
        logits = (rng.standard_normal((batch, beams, vocab)) * 3).astype(dtype)
        want = ref.select(logits, scores, beams, ended, eos)
        got = {name: t.to_numpy() for name, t in select.eval(up(logits), up(scores), ended=up(ended)).items()}
        for name in ("parents", "tokens", "ended"):
            np.testing.assert_array_equal(got[name], want[name], err_msg=f"{name}, turn {turn}")
        scores, ended, parents = got["scores"], got["ended"], got["parents"].reshape(-1)
        cache.reorder(up(parents))
        assert cache.missing() == 0
        plain.reorder(parents)
        _held(cache)
        step(1 - ended.reshape(-1).astype(int) * (turn % 2), 1 + turn % 3)
    gone = np.where(np.arange(n) < n // 2, -1, np.arange(n))
    cache.reorder(up(gone.astype(I32)))
    plain.reorder(gone)
    _held(cache)
    step(np.ones(n, int), 1)
    cache.reorder(up(np.full(n, -1, I32)))
    assert cache.free() == cache.n_pages and not cache.lens().any()


def test_a_cache_that_is_full_goes_on_when_pages_come_back(rt):
    rng, page, d = np.random.default_rng(0), 16, 64
    cache = ta.PagedKvCache(6, page, 1, d, 4, 64, F16)
    rows = lambda n: (up(rng.standard_normal((n, 1, d)).astype(F16)), up(rng.standard_normal((n, 1, d)).astype(F16)))  # noqa: E731
    cache.plan(up(np.array([33, 20, 0, 0], I32)), 53)
    cache.append(0, *rows(53))
    assert cache.refused() == 0 and cache.free() == 1
    cache.plan(up(np.array([0, 0, 17, 5], I32)), 22)       # two pages, and one for a later one that is not left either
    cache.append(0, *rows(22))
    assert cache.refused() == 2 and cache.free() == 1 and cache.lens().tolist() == [33, 20, 0, 0]
    assert (cache.slots.to_numpy() == -1).all()
    q = up(rng.standard_normal((4, 2, 1, d)).astype(F16))
    out = cache.attend(0, q).to_numpy()
    assert np.isfinite(out).all() and not out[2:].any()
    cache.reorder(up(np.array([0, 0, -1, -1], I32)))       # the second goes on from the first: one page for its copy
    assert cache.missing() == 0 and cache.free() == 2 and cache.lens().tolist() == [33, 33, 0, 0]
    cache.reorder(up(np.array([0, 0, 0, 0], I32)))
    assert cache.missing() == 1 and cache.lens().tolist() == [33, 33, 0, 0]    # of three copies one has no page: nothing changes
    cache.reorder(up(np.array([-1, 1, -1, -1], I32)))
    assert cache.missing() == 0 and cache.free() == 3
    cache.plan(up(np.array([0, 0, 17, 5], I32)), 22)
    assert cache.refused() == 0 and cache.lens().tolist() == [0, 33, 17, 5]
    _held(cache)
    with pytest.raises(ta.TractRocmError):
        ta.PagedKvCache(6, page, 1, d, 4, 64, F16).append(0, *rows(3))
    with pytest.raises(ta.TractRocmError):
        ta.PagedKvCache(0, page, 1, d, 4, 64, F16)


# ---- streams, threads, graphs ---------------------------------------------------------------------------------------------


def _calls(seed, dtype=F16):
    """name -> (call(stream), outputs): each with outputs and, where one is taken, an operator and a workspace of its own."""
    rng, calls = np.random.default_rng(seed), {}
    for name, lens, hq, hkv, sq, d, page in (("few", [3000, 700], 8, 2, 1, 128, 16), ("many", rng.integers(0, 400, 300), 4, 1, 2, 64, 32), ("any", [50, 90], 4, 2, 1, 40, 5)):
        held = -(-np.asarray(lens) // page)
        n_pages, width = int(held.sum()) + 1, int(held.max())
        table, at = np.full((len(lens), width), -1, I32), 0
        for i, h in enumerate(held):
            table[i, :h] = np.arange(at, at + h)
            at += h
        q, k, v = (up((rng.standard_normal(s) * 2).astype(dtype)) for s in ((len(lens), hq, sq, d), (n_pages, hkv, page, d), (n_pages, hkv, page, d)))
        out, op, a = ta.DeviceTensor(q.shape, dtype), ta.PagedSdpa(), (q, k, v, up(table), up(np.asarray(lens, I32)))
        calls[name] = (lambda stream, op=op, a=a, out=out: op.eval(*a, stream=stream, out=out)), [out]
    for name, batch, beams, vocab in (("one", 1, 4, 30000), ("batch", 20, 4, 50001)):
        x, s = up((rng.standard_normal((batch, beams, vocab)) * 3).astype(dtype)), up(-rng.random((batch, beams)).astype(F32))
        out = {"scores": ta.DeviceTensor((batch, 8), F32), **{y: ta.DeviceTensor((batch, 8), I32) for y in ("parents", "tokens", "ended")}}
        op = ta.BeamSelect(8, eos=3)
        calls[name] = (lambda stream, op=op, x=x, s=s, out=out: op.eval(x, s, stream=stream, out=out)), list(out.values())
    return calls


def _bytes(outs, stream=None):
    return [o.to_numpy(stream).tobytes() for o in outs]


def _scrub(outs):
    for o in outs:
        a = np.full(o.shape, -77, o.dtype)
        ta._lib.call("trocm_h2d", o.ptr, a.ctypes.data_as(C.c_void_p), o.nbytes, None)
    ta.synchronize()


def _want(seed, dtype=F16):
    want = {}
    for name, (call, outs) in _calls(seed, dtype).items():
        call(None)
        want[name] = _bytes(outs)
    ta.synchronize()
    return want


@pytest.mark.parametrize("dtype", [F16, F32])
def test_two_streams_at_once(rt, dtype):
    want, sides = _want(1, dtype), [(_calls(1, dtype), ta.Stream()) for _ in range(2)]
    for _ in range(5):
        for calls, stream in sides:
            for call, _ in calls.values():
                call(stream)
    for calls, stream in sides:
        for name, (_, outs) in calls.items():
            assert _bytes(outs, stream) == want[name], name


def test_threads_with_streams_of_their_own(rt):
    want, wrong = _want(2), []

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


class Graph:
    """What `record` queues on the stream, to be replayed."""

    def __init__(self, stream, record):
        self.hip = C.CDLL("libamdhip64.so")
        self.handle = stream.handle if isinstance(stream.handle, C.c_void_p) else C.c_void_p(stream.handle)
        self.stream, self.graph, self.run = stream, C.c_void_p(), C.c_void_p()
        self.ok(self.hip.hipStreamBeginCapture(self.handle, C.c_int(1)))
        record()
        self.ok(self.hip.hipStreamEndCapture(self.handle, C.byref(self.graph)))
        self.ok(self.hip.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, C.c_size_t(0)))

    @staticmethod
    def ok(rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.run, self.handle))
        self.stream.synchronize()

    def close(self):
        self.ok(self.hip.hipGraphExecDestroy(self.run))
        self.ok(self.hip.hipGraphDestroy(self.graph))


def test_captured_and_replayed_with_a_shared_workspace(rt):
    """Two graphs of the same calls, replayed in turn between eager calls of the same operators (one stream, one workspace each)."""
    want, calls, stream = _want(3), _calls(3), ta.Stream()
    for call, _ in calls.values():
        call(stream)
    stream.synchronize()
    graphs = [Graph(stream, lambda: [call(stream) for call, _ in calls.values()]) for _ in range(2)]
    for turn in range(6):
        for _, outs in calls.values():
            _scrub(outs)
        graphs[turn % 2].replay()
        for name, (_, outs) in calls.items():
            assert _bytes(outs, stream) == want[name], f"replay {turn}: {name}"
        for name, (call, outs) in calls.items():
            _scrub(outs)
            call(stream)
            assert _bytes(outs, stream) == want[name], f"eager call after replay {turn}: {name}"
    for g in graphs:
        g.close()


@pytest.mark.parametrize("dtype,d,page", [(F16, 128, 16), (F32, 64, 16), (F16, 24, 3)])
def test_recorded_steps_go_on_by_themselves(rt, dtype, d, page):
    """Two steps, their plans, appends, attention and a reorder between them, recorded once: every replay starts where the last one ended, and
    leaves what the same steps leave that are queued one by one."""
    rng, n, hq, hkv, stream = np.random.default_rng(11), 5, 4, 2, ta.Stream()
    caches = [ta.PagedKvCache(60, page, hkv, d, n, 20 * page, dtype) for _ in range(2)]
    new = [up(np.array(x, I32)) for x in ([1, 1, 0, 1, 3], [2, 1, 1, 1, 0])]
    parents = [up(np.array(x, I32)) for x in ([0, 0, 2, 3, 4], [0, 1, 2, 3, 4])]
    tokens = [6, 5]
    k, v = ([up(rng.standard_normal((t, hkv, d)).astype(dtype)) for t in tokens] for _ in range(2))
    q = [up(rng.standard_normal((n, hq, 1, d)).astype(dtype)) for _ in range(2)]
    out = [[ta.DeviceTensor((n, hq, 1, d), dtype) for _ in range(2)] for _ in range(2)]
    plans = [[{x: ta.DeviceTensor((s,), I32) for x, s in (("starts", n + 1), ("slots", t), ("positions", t))} for t in tokens] for _ in range(2)]

    def steps(side):
        c = caches[side]
        for i in range(2):
            c.plan(new[i], tokens[i], stream=stream, out=plans[side][i])
            c.append(0, k[i], v[i], stream=stream)
            c.attend(0, q[i], stream=stream, out=out[side][i])
            c.reorder(parents[i], stream=stream)

    steps(0), steps(1)     # (workspaces, and pages to begin with)
    stream.synchronize()
    graph = Graph(stream, lambda: steps(1))
    for turn in range(6):
        steps(0)
        stream.synchronize()
        graph.replay()
        assert caches[0].lens(stream).tolist() == caches[1].lens(stream).tolist()
        assert caches[0].lens(stream).max() > 2 * turn
        for name in ("table", "refs", "free", "count"):
            np.testing.assert_array_equal(caches[0]._now(name).to_numpy(stream), caches[1]._now(name).to_numpy(stream), err_msg=name)
        for i in range(2):
            a, b = out[0][i].to_numpy(stream), out[1][i].to_numpy(stream)
            assert np.isfinite(a).all() and a.tobytes() == b.tobytes(), (turn, i)
    graph.close()


def test_replayed_after_a_larger_call(rt):
    """Recorded calls are replayed after their operators took larger shapes: the workspace that a graph knows stays, and the results too."""
    rng, stream, op, select = np.random.default_rng(12), ta.Stream(), ta.PagedSdpa(), ta.BeamSelect(4)

    def calls(n):
        k, v, q = (up(rng.standard_normal(s).astype(F16)) for s in ((n * 64, 1, 16, 64), (n * 64, 1, 16, 64), (n, 4, 1, 64)))
        table, lens, out = up(np.arange(n * 64, dtype=I32).reshape(n, 64)), up(np.full(n, 1000, I32)), ta.DeviceTensor((n, 4, 1, 64), F16)
        x, s, chosen = up(rng.standard_normal((n, 2, 9000)).astype(F32)), up(np.zeros((n, 2), F32)), {"scores": ta.DeviceTensor((n, 4), F32)}
        chosen.update({y: ta.DeviceTensor((n, 4), I32) for y in ("parents", "tokens", "ended")})
        return lambda: (op.eval(q, k, v, table, lens, stream=stream, out=out), select.eval(x, s, stream=stream, out=chosen)), [out, *chosen.values()]

    small, outs = calls(2)
    small()
    want = _bytes(outs, stream)
    graph = Graph(stream, small)
    for n in (1, 40, 300):
        larger, _ = calls(n)
        for _ in range(2):
            larger()
            _scrub(outs)
            graph.replay()
            assert _bytes(outs, stream) == want, n
        _scrub(outs)
        small()
        assert _bytes(outs, stream) == want, n
    graph.close()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_workspace_for_operators_in_turn(rt, dtype):
    """The dense and the paged attention and beam search's choice leave a workspace ready for each other."""
    rng = np.random.default_rng(4)
    b, hq, hkv, t, d, page = 6, 8, 2, 2560, 128, 16
    q, k, v = (up(rng.standard_normal(s).astype(dtype)) for s in ((b, hq, 1, d), (b, hkv, t, d), (b, hkv, t, d)))
    pages = [up(np.ascontiguousarray(x.to_numpy().reshape(b, hkv, t // page, page, d).transpose(0, 2, 1, 3, 4).reshape(-1, hkv, page, d))) for x in (k, v)]
    table, lens = up(np.arange(b * t // page, dtype=I32).reshape(b, -1)), up(np.full(b, t, I32))
    out = [ta.DeviceTensor((b, hq, 1, d), dtype) for _ in range(2)]
    x, s = up((rng.standard_normal((b, 4, 20000)) * 3).astype(dtype)), up(np.zeros((b, 4), F32))
    chosen = {"scores": ta.DeviceTensor((b, 4), F32), **{y: ta.DeviceTensor((b, 4), I32) for y in ("parents", "tokens", "ended")}}
    sizes = [C.c_size_t() for _ in range(2)]
    ta._lib.call("trocm_sdpa_paged_workspace_bytes", b, hq, hkv, 1, d, C.byref(sizes[0]))
    ta._lib.call("trocm_beam_select_workspace_bytes", b, 4, 20000, 4, C.byref(sizes[1]))
    ws = ta.Workspace(b, hq, 1, d, nbytes=max(ta.Workspace.bytes_for(b, hq, 1, d), *(z.value for z in sizes)))
    code, nan = 0 if dtype == F32 else 1, float("nan")
    steps = {
        "dense": (lambda: ta._lib.call("trocm_sdpa", q.ptr, k.ptr, v.ptr, None, out[0].ptr, code, b, hq, hkv, 1, t, d, None, 0, 0, nan, 1, ws.ptr, ws.nbytes, None), [out[0]]),
        "paged": (lambda: ta._lib.call("trocm_sdpa_paged", q.ptr, code, b, hq, hkv, 1, d, pages[0].ptr, pages[1].ptr, b * t // page, page, None, table.ptr, t // page, lens.ptr, out[1].ptr, nan, 1,
                                       ws.ptr, ws.nbytes, None), [out[1]]),
        "select": (lambda: ta._lib.call("trocm_beam_select", x.ptr, code, b, 4, 20000, 0, s.ptr, None, -1, 4, chosen["scores"].ptr, chosen["parents"].ptr, chosen["tokens"].ptr,
                                        chosen["ended"].ptr, ws.ptr, ws.nbytes, None), list(chosen.values())),
    }
    want = {}
    for name, (step, outs) in steps.items():
        step()
        want[name] = _bytes(outs)
    for name in ("dense", "paged", "dense", "select", "paged", "select", "dense", "dense", "select", "select", "paged", "paged") * 2:
        step, outs = steps[name]
        _scrub(outs)
        step()
        assert _bytes(outs) == want[name], name
    exact = ref.attend(q.to_numpy(), *(y.to_numpy() for y in (*pages, table, lens)))
    for small in (0, 100, 1 << 16):     # too little for the fast kernel, and for the choice
        _scrub([out[1]])
        ta._lib.call("trocm_sdpa_paged", q.ptr, code, b, hq, hkv, 1, d, pages[0].ptr, pages[1].ptr, b * t // page, page, None, table.ptr, t // page, lens.ptr, out[1].ptr, nan, 1,
                     ws.ptr if small else None, small, None)
        attention_ref.assert_within(out[1].to_numpy(), *exact)
        with pytest.raises(ta.TractRocmError, match="workspace"):
            ta._lib.call("trocm_beam_select", x.ptr, code, b, 4, 20000, 0, s.ptr, None, -1, 4, chosen["scores"].ptr, chosen["parents"].ptr, chosen["tokens"].ptr, chosen["ended"].ptr,
                         ws.ptr, small, None)
