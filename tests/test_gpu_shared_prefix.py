"""Attention of sequences that share a prefix, over tensors and over caches, against 64 bits."""
import ctypes as C

import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, norm_rope, shared
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


def _case(rng, lens, hq, hkv, p, sq, d, dtype, room=None):
    n, room = len(lens), max(1, max(lens)) if room is None else room
    q = _rows(rng, (n, hq, sq, d), dtype, 2.0)
    pk, pv = (_rows(rng, (1, hkv, p, d), dtype) for _ in range(2))
    k, v = (_rows(rng, (n, hkv, room, d), dtype) for _ in range(2))
    for i, length in enumerate(lens):     # what lies behind a sequence's last key is never read
        k[i, :, length:], v[i, :, length:] = np.nan, np.inf
    return q, pk, pv, k, v


def _want(q, pk, pv, k, v, lens, **kw):
    return shared(q, pk[0], pv[0], [t[:, :n] for t, n in zip(k, lens)], [t[:, :n] for t, n in zip(v, lens)], **kw)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,hq,hkv,p,sq,d", [
    ([1], 8, 2, 1, 1, 64), ([0, 0, 0], 4, 1, 77, 1, 128), ([3, 0, 40], 14, 2, 777, 1, 64), ([5, 33, 64, 1], 4, 4, 130, 1, 128),
    ([100, 1, 31, 32, 33], 8, 2, 0, 1, 64), ([0, 7], 4, 2, 0, 1, 128), ([9, 200, 17], 8, 8, 515, 1, 64),
    (list(range(0, 90, 3)), 16, 2, 1000, 1, 128), ([600, 2], 32, 1, 64, 1, 64),
    ([4, 20, 3], 6, 2, 300, 4, 128), ([2, 50], 8, 1, 33, 9, 64),        # several queries each; fewer own keys than queries
    ([5, 2], 6, 3, 40, 1, 80), ([3, 4, 0], 2, 1, 9, 2, 200), ([1, 2], 2, 2, 5, 1, 7)])   # head sizes without a kernel of their own
def test_over_tensors(rt, dtype, lens, hq, hkv, p, sq, d):
    rng = np.random.default_rng(1)
    q, pk, pv, k, v = _case(rng, lens, hq, hkv, max(p, 1), sq, d, dtype)
    op = ta.SharedPrefixSdpa()
    for _ in range(2):   # the workspace is ready for the next call
        got = op.eval(q, pk, pv, k, v, lens, prefix_len=p)
        assert_within(got.to_numpy(), *_want(q, pk[:, :, :p], pv[:, :, :p], k, v, lens))
    if p == 0:
        for i, n in enumerate(lens):
            assert n or not got.to_numpy()[i].any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,hq,hkv,p,longest,d", [(64, 8, 2, 2500, 130, 128), (130, 14, 2, 300, 40, 64), (750, 2, 1, 100, 12, 64), (3, 64, 8, 5000, 900, 64)])
def test_many_and_long(rt, dtype, n, hq, hkv, p, longest, d):
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, longest, n, endpoint=True)]
    case = _case(rng, lens, hq, hkv, p, 1, d, dtype)
    got = ta.SharedPrefixSdpa().eval(*case, lens)
    assert_within(got.to_numpy(), *_want(*case, lens))


@pytest.mark.parametrize("dtype,n,hq,hkv,p,longest,d", [
    (F16, 3, 32, 8, 30000, 50, 128), (F16, 10, 32, 8, 27000, 90, 128), (F16, 64, 32, 8, 6000, 700, 128), (F16, 1, 64, 8, 60000, 9, 64), (F16, 40, 64, 8, 6000, 2800, 64),
    (F32, 3, 32, 8, 15000, 50, 128), (F32, 20, 8, 8, 2000, 900, 64), (F32, 70, 32, 8, 800, 500, 128)])
def test_more_keys_than_caches_hold(rt, dtype, n, hq, hkv, p, longest, d):
    """100 MB of keys and more; some heads of some sequences against 64 bits, all of a second call against the first."""
    rng = np.random.default_rng(21)
    lens = [int(x) for x in rng.integers(longest // 2, longest, n, endpoint=True)]
    q, pk, pv, k, v = case = _case(rng, lens, hq, hkv, p, 1, d, dtype)
    device = [ta.DeviceTensor.from_numpy(t) for t in case]
    op = ta.SharedPrefixSdpa()
    got = op.eval(*device, lens).to_numpy()
    for i, h in zip(rng.integers(0, n, 12), rng.integers(0, hq, 12)):
        g = h * hkv // hq
        want = shared(q[i : i + 1, h : h + 1], pk[0, g : g + 1], pv[0, g : g + 1], [k[i, g : g + 1, : lens[i]]], [v[i, g : g + 1, : lens[i]]])
        assert_within(got[i : i + 1, h : h + 1], *want, what=f"sequence {i}, head {h}")
    assert op.eval(*device, lens).to_numpy().tobytes() == got.tobytes()


@pytest.mark.parametrize("d", [64, 128])
def test_prefixes_whose_scores_rise_late(rt, d):
    rng = np.random.default_rng(24)
    n, hq, hkv, p = 40, 32, 4, 4000
    lens = [int(x) for x in rng.integers(0, 90, n)]
    q, pk, pv, k, v = _case(rng, lens, hq, hkv, p, 1, d, F16)
    q = (q * 15).astype(F16)
    for growth in (np.linspace(0.02, 1.5, p), np.linspace(1.5, 0.02, p), np.zeros(p), np.where(np.arange(p) % 1331 == 1330, 3.0, 0.05)):
        kk = (pk * growth[None, None, :, None]).astype(F16)
        got = ta.SharedPrefixSdpa().eval(q, kk, pv, k, v, lens).to_numpy()
        some = list(range(0, n, 13))
        assert_within(got[some], *_want(q[some], kk, pv, [k[i] for i in some], [v[i] for i in some], [lens[i] for i in some]))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_not_causal_scale_strides_and_small_workspaces(rt, dtype):
    rng = np.random.default_rng(3)
    lens, hq, hkv, p, sq, d = [40, 7, 0], 8, 2, 200, 3, 64
    q, pk, pv, k, v = _case(rng, lens, hq, hkv, p, sq, d, dtype)
    got = ta.SharedPrefixSdpa(scale=0.05, is_causal=False).eval(q, pk, pv, k, v, lens)
    assert_within(got.to_numpy(), *_want(q, pk, pv, k, v, lens, scale=0.05, causal=False))
    # a prefix laid out by tokens, a base that no 16-byte access fits, no workspace
    want = _want(q, pk, pv, k, v, lens)
    es = np.dtype(dtype).itemsize
    by_token = [np.ascontiguousarray(t[0].transpose(1, 0, 2)) for t in (pk, pv)]
    for shift, ws_bytes in ((0, 0), (1, 0), (0, 1 << 16), (0, 400 << 10)):
        flat = [ta.DeviceTensor.from_numpy(np.concatenate([np.zeros(shift, dtype), t.reshape(-1)])) for t in by_token]
        dq, dk, dv = (ta.DeviceTensor.from_numpy(t) for t in (q, k, v))
        out = ta.DeviceTensor(q.shape, dtype)
        ws = ta.Workspace(1, 1, 1, 64, nbytes=ws_bytes) if ws_bytes else None
        room = k.shape[2]
        ta._lib.call("trocm_sdpa_shared_prefix", dq.ptr, 0 if dtype == F32 else 1, 3, hq, hkv, sq, d, flat[0].ptr.value + shift * es, flat[1].ptr.value + shift * es, p,
                     (C.c_int64 * 2)(d, hkv * d), dk.ptr, dv.ptr, (C.c_int64 * 3)(hkv * room * d, room * d, d), (C.c_int64 * 3)(*lens), out.ptr,
                     float("nan"), 1, ws.ptr if ws else None, ws_bytes, None)
        assert_within(out.to_numpy(), *want, what=f"shift {shift}, workspace {ws_bytes}")


@pytest.mark.parametrize("dtype,hq,hkv,d,n_seq", [(F16, 8, 2, 128, 5), (F32, 6, 2, 64, 3), (F16, 4, 4, 96, 2), (F16, 8, 1, 64, 100)])
def test_steps_over_caches(rt, dtype, hq, hkv, d, n_seq):
    """Steps of one and of several tokens: the caches hold what was appended, the output attends to it."""
    rng = np.random.default_rng(4)
    p = 150
    pk, pv = (_rows(rng, (1, hkv, p, d), dtype) for _ in range(2))
    prefix = [ta.InPlaceKvCache(2) for _ in range(2)]
    prefix[0].push(pk), prefix[1].push(pv)
    ks, vs = ([ta.InPlaceKvCache(2) for _ in range(n_seq)] for _ in range(2))
    own_k, own_v = ([np.zeros((hkv, 0, d), dtype) for _ in range(n_seq)] for _ in range(2))
    for i in range(0, n_seq, 2):   # half of the sequences have begun before
        n = 1 + 13 * i % 37
        own_k[i], own_v[i] = _rows(rng, (hkv, n, d), dtype), _rows(rng, (hkv, n, d), dtype)
        ks[i].push(own_k[i][None]), vs[i].push(own_v[i][None])
    ws = ta.Workspace(n_seq, hq, 4, d, nbytes=ta.Workspace.shared_bytes_for(n_seq, hq, 4, d))
    for sq in (1, 1, 4, 1):
        q = _rows(rng, (n_seq, hq, sq, d), dtype, 2.0)
        kn, vn = (_rows(rng, (n_seq, hkv, sq, d), dtype) for _ in range(2))
        dq, dk, dv = (ta.DeviceTensor.from_numpy(t) for t in (q, kn, vn))
        got = ta.inplace_kv_sdpa_eval_shared(dq, dk, dv, *prefix, ks, vs, workspace=ws).to_numpy()
        own_k, own_v = ([np.concatenate([o, t], axis=1) for o, t in zip(own, new)] for own, new in ((own_k, kn), (own_v, vn)))
        assert_within(got, *shared(q, pk[0], pv[0], own_k, own_v))
        for c, o in zip(ks + vs, own_k + own_v):
            assert c.valid_contiguous().tobytes() == o[None].tobytes()
        again = ta.inplace_kv_sdpa_eval_shared(dq, None, None, *prefix, ks, vs, workspace=ws).to_numpy()
        assert again.tobytes() == got.tobytes()
    assert prefix[0].valid_contiguous().tobytes() == pk.tobytes() and prefix[0].len() == p


def test_norm_rope_then_shared_step(rt):
    """Two layers' worth of a decode step as it is used: norms and rotation, then the step over the shared prefix, all queued before anything is read."""
    rng = np.random.default_rng(5)
    n_seq, hq, hkv, d, p = 6, 8, 2, 128, 300
    stream = ta.Stream()
    angle = (p + np.arange(n_seq))[:, None, None, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    cos, sin = (f(np.concatenate([angle, angle], axis=-1)).astype(F16) for f in (np.cos, np.sin))
    layers = []
    for _ in range(2):
        pk, pv = (_rows(rng, (1, hkv, p, d), F16) for _ in range(2))
        prefix = [ta.InPlaceKvCache(2) for _ in range(2)]
        prefix[0].push(pk, stream=stream), prefix[1].push(pv, stream=stream)
        q, k, v = (_rows(rng, (n_seq, h, 1, d), F16) for h in (hq, hkv, hkv))
        layers.append((pk, pv, prefix, q, k, v, [ta.InPlaceKvCache(2) for _ in range(n_seq)], [ta.InPlaceKvCache(2) for _ in range(n_seq)]))
    dc, ds = (ta.DeviceTensor.from_numpy(t) for t in (cos, sin))
    op, outs, keep = ta.QkNormRope(1e-6), [], []
    ws = ta.Workspace(n_seq, hq, 1, d, nbytes=ta.Workspace.shared_bytes_for(n_seq, hq, 1, d))
    for pk, pv, prefix, q, k, v, ks, vs in layers:
        dq, dk, dv = (ta.DeviceTensor.from_numpy(t) for t in (q, k, v))
        nq, nk = op.eval(dq, dk, None, None, dc, ds, stream=stream)
        outs.append((ta.inplace_kv_sdpa_eval_shared(nq, nk, dv, *prefix, ks, vs, workspace=ws, stream=stream), nq, nk))
        keep += [dq, dk, dv]
    for (out, nq, nk), (pk, pv, prefix, q, k, v, ks, vs) in zip(outs, layers):
        gq, gk = nq.to_numpy(stream), nk.to_numpy(stream)
        assert_within(gq, *norm_rope(q, None, cos, sin, 1e-6))
        assert_within(gk, *norm_rope(k, None, cos, sin, 1e-6))
        assert_within(out.to_numpy(stream), *shared(gq, pk[0], pv[0], list(gk), list(v)))


def test_refusals_leave_the_caches(rt):
    rng = np.random.default_rng(6)
    hq, hkv, d = 4, 2, 64
    prefix = [ta.InPlaceKvCache(2) for _ in range(2)]
    for c in prefix:
        c.push(_rows(rng, (1, hkv, 20, d), F16))
    ks, vs = ([ta.InPlaceKvCache(2) for _ in range(2)] for _ in range(2))
    q = ta.DeviceTensor.from_numpy(_rows(rng, (2, hq, 1, d), F16))
    new = ta.DeviceTensor.from_numpy(_rows(rng, (2, hkv, 1, d), F16))
    ta.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, ks, vs)
    with pytest.raises(ta.TractRocmError, match="all different"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, [ks[0], ks[0]], vs)
    with pytest.raises(ta.TractRocmError, match="all different"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, [ks[0], prefix[0]], [vs[0], prefix[1]])
    with pytest.raises(ta.TractRocmError, match="out overlaps"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, ks, vs, out=q)
    with pytest.raises(ta.TractRocmError, match="k_new / v_new"):
        ta.inplace_kv_sdpa_eval_shared(q, new, None, *prefix, ks, vs)
    quant = [ta.InPlaceKvCache(2, ta.Q8_0) for _ in range(2)]
    for c in quant:
        c.push(_rows(rng, (1, hkv, 20, d), F16))
    with pytest.raises(ta.TractRocmError, match="block-quantised"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *quant, ks, vs)
    window = [ta.WindowKvCache(2, 8) for _ in range(2)]
    for c in window:
        c.push(_rows(rng, (1, hkv, 1, d), F16))
    with pytest.raises(ta.TractRocmError, match="ring buffers"):
        ta.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, [ks[0], window[0]], [vs[0], window[1]])
    assert [c.len() for c in ks + vs + prefix] == [1, 1, 1, 1, 20, 20]
    # two sequences that only read may share a cache
    a = ta.inplace_kv_sdpa_eval_shared(q, None, None, *prefix, [ks[0], ks[0]], [vs[0], vs[0]]).to_numpy()
    assert np.isfinite(a).all()
