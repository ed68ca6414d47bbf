"""Attention with capped scores, distance slopes, documents and prefixes, against 64 bits."""
import ctypes as C
import itertools

import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, scored, shared
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


def _slopes(hq):
    return (2.0 ** (-8.0 * (np.arange(hq) + 1) / hq)).astype(F32)


def _packed(rng, b, t, docs):
    ends = np.sort(rng.integers(0, t, (b, docs - 1)), axis=1)
    return np.stack([np.searchsorted(e, np.arange(t), side="right") for e in ends]).astype(np.int32)


def _check(dtype, b, hq, hkv, n, t, d, cap=0.0, slopes=None, documents=None, prefix_lens=None, causal=True, scale=None, seed=0, big=4.0):
    rng = np.random.default_rng(seed)
    q, k, v = _rows(rng, (b, hq, n, d), dtype, big), _rows(rng, (b, hkv, t, d), dtype), _rows(rng, (b, hkv, t, d), dtype)
    op = ta.ScoredSdpa(scale, cap, causal)
    rules = dict(slopes=slopes, documents=documents, prefix_lens=prefix_lens)
    got = op.eval(q, k, v, **rules).to_numpy()
    assert_within(got, *scored(q, k, v, scale, cap, causal=causal, **rules))
    return got


SHAPES = [(1, 4, 1, 1, 1, 64), (2, 8, 2, 1, 300, 128), (1, 14, 2, 3, 65, 64), (1, 4, 4, 33, 33, 128), (2, 4, 2, 70, 201, 64),
          (1, 8, 1, 129, 129, 128), (1, 3, 1, 5, 40, 96), (1, 2, 2, 4, 11, 8), (1, 2, 1, 300, 300, 64), (1, 32, 1, 1, 1000, 64)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rules", list(itertools.product([False, True], repeat=4)), ids=lambda r: "".join("csdp"[i] if x else "-" for i, x in enumerate(r)))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_rule_and_shape(rt, dtype, rules, shape):
    b, hq, hkv, n, t, d = shape
    cap, slopes, documents, prefix = rules
    rng = np.random.default_rng(9)
    _check(dtype, *shape, cap=15.0 if cap else 0.0, slopes=_slopes(hq) if slopes else None, documents=_packed(rng, b, t, 4) if documents else None,
           prefix_lens=rng.integers(0, t, b, endpoint=True).astype(np.int32) if prefix else None)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("b,hq,hkv,n,t,d", [(1, 8, 2, 500, 500, 128), (1, 4, 2, 260, 1300, 64), (2, 2, 2, 700, 700, 64), (3, 16, 2, 1, 5000, 128), (1, 6, 1, 11, 3000, 128),
                                            (1, 7, 1, 640, 641, 64)])
def test_longer(rt, dtype, b, hq, hkv, n, t, d):
    rng = np.random.default_rng(10)
    _check(dtype, b, hq, hkv, n, t, d, cap=30.0)
    _check(dtype, b, hq, hkv, n, t, d, slopes=_slopes(hq), documents=_packed(rng, b, t, 7))
    _check(dtype, b, hq, hkv, n, t, d, cap=20.0, prefix_lens=np.array([t // 3] * b, np.int32))


@pytest.mark.parametrize("b,hq,hkv,n,t,d", [(1, 32, 8, 1000, 1000, 128), (3, 28, 4, 1000, 1040, 64), (1, 64, 8, 777, 800, 64)])
def test_enough_rows_for_every_compute_unit(rt, b, hq, hkv, n, t, d):
    """128 rows per workgroup, its tiles taken by one group of waves or by two in turn."""
    rng = np.random.default_rng(15)
    _check(F16, b, hq, hkv, n, t, d, cap=30.0)
    _check(F16, b, hq, hkv, n, t, d, cap=20.0, slopes=_slopes(hq), documents=_packed(rng, b, t, 5), prefix_lens=np.full(b, t // 4, np.int32))


@pytest.mark.parametrize("rules", list(itertools.product([False, True], repeat=3)), ids=lambda r: "".join("csd"[i] if x else "-" for i, x in enumerate(r)))
@pytest.mark.parametrize("shape", [(1, 32, 8, 1000, 1000, 128), (2, 28, 4, 1000, 1040, 64), (4, 32, 32, 300, 300, 128), (8, 64, 32, 300, 310, 64)], ids=str)
def test_every_rule_where_rows_fill_the_card(rt, rules, shape):
    """Head sizes 128 and 64, one group of waves per workgroup and two; keys before the queries, of the first of them none for some rows."""
    b, hq, hkv, n, t, d = shape
    cap, slopes, documents = rules
    _check(F16, *shape, cap=25.0 if cap else 0.0, slopes=_slopes(hq) if slopes else None, documents=_packed(np.random.default_rng(16), b, t, 3) if documents else None)


def test_unusual_scales_where_rows_fill_the_card(rt):
    shape = (1, 32, 8, 1000, 1000, 128)
    _check(F16, *shape, slopes=_slopes(32), scale=-0.05)
    _check(F16, *shape, scale=0.0)
    _check(F16, *shape, cap=10.0, scale=-0.05, slopes=_slopes(32))
    _check(F16, *shape, cap=1e-9, slopes=_slopes(32))
    _check(F16, *shape, slopes=_slopes(32), scale=1e-9)
    _check(F16, 1, 32, 8, 1000, 900, 128, cap=10.0)               # fewer keys than queries
    _check(F16, 1, 32, 8, 1000, 1000, 128, slopes=_slopes(32), causal=False)


@pytest.mark.parametrize("dtype,b,hq,hkv,t,d", [(F16, 4, 32, 8, 8200, 128), (F16, 7, 16, 8, 8200, 64), (F32, 2, 32, 8, 8200, 128), (F32, 4, 8, 8, 8200, 64)])
def test_single_tokens_over_more_keys_than_caches_hold(rt, dtype, b, hq, hkv, t, d):
    rng = np.random.default_rng(22)
    q, k, v = _rows(rng, (b, hq, 1, d), dtype, 4.0), _rows(rng, (b, hkv, t, d), dtype), _rows(rng, (b, hkv, t, d), dtype)
    ids = _packed(rng, b, t, 3)
    device = [ta.DeviceTensor.from_numpy(x) for x in (q, k, v)]
    for rules in ({}, {"slopes": _slopes(hq) * 1e-2}, {"documents": ids}):
        got = ta.ScoredSdpa(softcap=30.0).eval(*device, **rules).to_numpy()
        for i, h in zip(rng.integers(0, b, 8), rng.integers(0, hq, 8)):
            some = {x: y[i : i + 1] if x == "documents" else y[h : h + 1] for x, y in rules.items()}
            g = h * hkv // hq
            want = scored(q[i : i + 1, h : h + 1], k[i : i + 1, g : g + 1], v[i : i + 1, g : g + 1], cap=30.0, **some)
            assert_within(got[i : i + 1, h : h + 1], *want, what=f"{list(rules)}, batch {i}, head {h}")


@pytest.mark.parametrize("d", [64, 128])
def test_rows_whose_maximum_rises_late_and_rows_that_are_not_numbers(rt, d):
    """Scores that grow along the keys and against them, far apart, all alike; a query row of NaN is the only one that shows it."""
    rng = np.random.default_rng(23)
    b, hq, hkv, n = 1, 64, 8, 1000
    q, k, v = _rows(rng, (b, hq, n, d), F16, 40.0), _rows(rng, (b, hkv, n, d), F16), _rows(rng, (b, hkv, n, d), F16)
    for growth in (np.linspace(0.02, 1.5, n), np.linspace(1.5, 0.02, n), np.zeros(n), np.where(np.arange(n) % 331 == 330, 3.0, 0.05)):
        kk = (k * growth[None, None, :, None]).astype(F16)
        for rules in ({}, {"slopes": _slopes(hq)}, {"documents": _packed(rng, b, n, 4)}):
            got = ta.ScoredSdpa().eval(q, kk, v, **rules).to_numpy()
            assert_within(got[:, 3:40:9], *scored(q[:, 3:40:9], kk[:, [3 * hkv // hq, 12 * hkv // hq, 21 * hkv // hq, 30 * hkv // hq, 39 * hkv // hq]],
                                                  v[:, [3 * hkv // hq, 12 * hkv // hq, 21 * hkv // hq, 30 * hkv // hq, 39 * hkv // hq]],
                                                  **{x: y[3:40:9] if x == "slopes" else y for x, y in rules.items()}))
    plain = ta.ScoredSdpa(softcap=30.0).eval(q, k, v).to_numpy()
    q[0, 5, 700] = np.nan
    got = ta.ScoredSdpa(softcap=30.0).eval(q, k, v).to_numpy()
    assert np.isnan(got[0, 5, 700]).all()
    got[0, 5, 700] = plain[0, 5, 700]
    assert got.tobytes() == plain.tobytes()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_more_tiles_of_rows_than_one_axis_of_a_grid_has_places(rt, dtype):
    """Over a few keys, where every row is a row of its own in 64 bits too: those at both ends and about tile 65535 of 16 and of 32 rows."""
    rng = np.random.default_rng(19)
    hq, n, t, d = 16, 132000, 20, 64
    q, k, v = _rows(rng, (1, hq, n, d), dtype), _rows(rng, (1, 1, t, d), dtype), _rows(rng, (1, 1, t, d), dtype)
    got = ta.ScoredSdpa(softcap=5.0, is_causal=False).eval(q, k, v).to_numpy()
    at = np.r_[0:40, 65500:65570, 131000:131140, n - 40 : n]
    assert_within(got[:, :, at], *scored(q[:, :, at], k, v, cap=5.0, causal=False))


@pytest.mark.parametrize("hq,hkv,n", [(64, 8, 1000), (4, 2, 3)])
def test_documents_over_very_many_keys(rt, hq, hkv, n):
    """More tiles of keys than are looked up beforehand: some rows of some heads against 64 bits."""
    rng = np.random.default_rng(17)
    t, d = 263000, 64
    q, k = _rows(rng, (1, hq, n, d), F16, 3.0), _rows(rng, (1, hkv, t, d), F16)
    v = np.ascontiguousarray(k[:, ::-1, ::-1])
    ids = rng.integers(0, 3, (1, t)).astype(np.int32)
    ids[0, 1000:1500], ids[0, t - 2] = -1, -1
    slopes = _slopes(hq) * 1e-4
    dq, dk, dv, di = (ta.DeviceTensor.from_numpy(x) for x in (q, k, v, ids))
    got = ta.ScoredSdpa(softcap=20.0).eval(dq, dk, dv, slopes=slopes, documents=di).to_numpy()
    for h, i in ((0, 0), (hq - 1, n - 1), (hq // 2, n - 2), (hq // 3, n // 2)):
        end = t - n + i + 1
        want = scored(q[:, h : h + 1, i : i + 1], *(x[:, h * hkv // hq][:, None, :end] for x in (k, v)), cap=20.0, slopes=slopes[h : h + 1], documents=ids[:, :end])
        assert_within(got[:, h : h + 1, i : i + 1], *want, what=f"head {h}, row {i}")


@pytest.mark.parametrize("dtype,n,d", [(F16, 1, 128), (F16, 70, 64), (F32, 1, 64), (F16, 2, 48)])
def test_keys_further_apart_than_32_bits(rt, dtype, n, d):
    """300 keys 2^24 bytes apart; over the same rows as a shared prefix too."""
    rng = np.random.default_rng(18)
    es, hq, hkv, t = np.dtype(dtype).itemsize, 4, 2, 300
    apart = 2**24 // es
    rows = _rows(rng, (t, 2, hkv, d), dtype)
    big = ta.DeviceTensor((t * apart,), dtype)
    for j in range(t):
        ta._lib.call("trocm_h2d", C.c_void_p(big.ptr.value + j * 2**24), rows[j].ctypes.data_as(C.c_void_p), rows[j].nbytes, None)
    ta.synchronize()
    k, v = (np.ascontiguousarray(rows[:, i].transpose(1, 0, 2))[None] for i in range(2))
    q = _rows(rng, (1, hq, n, d), dtype, 2.0)
    dq, out = ta.DeviceTensor.from_numpy(q), ta.DeviceTensor(q.shape, dtype)
    ws = ta.Workspace(1, hq, n, d, nbytes=ta.Workspace.shared_bytes_for(1, hq, n, d))
    code, v_at = 0 if dtype == F32 else 1, C.c_void_p(big.ptr.value + hkv * d * es)
    ta._lib.call("trocm_sdpa_scored", dq.ptr, big.ptr, v_at, out.ptr, code, 1, hq, hkv, n, t, d, (C.c_int64 * 3)(0, d, apart), float("nan"), 15.0, None, None, None, 1,
                 ws.ptr, ws.nbytes, None)
    assert_within(out.to_numpy(), *scored(q, k, v, cap=15.0))
    none = ta.DeviceTensor((1, hkv, 1, d), dtype)
    ta._lib.call("trocm_sdpa_shared_prefix", dq.ptr, code, 1, hq, hkv, n, d, big.ptr, v_at, t, (C.c_int64 * 2)(d, apart), none.ptr, none.ptr,
                 (C.c_int64 * 3)(hkv * d, d, d), (C.c_int64 * 1)(0), out.ptr, float("nan"), 1, ws.ptr, ws.nbytes, None)
    assert_within(out.to_numpy(), *shared(q, k[0], v[0], [k[0][:, :0]], [v[0][:, :0]]))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 9, 150])
def test_not_causal_and_scales(rt, dtype, n):
    rng = np.random.default_rng(11)
    _check(dtype, 2, 4, 2, n, 190, 64, cap=5.0, causal=False)
    _check(dtype, 2, 4, 2, n, 190, 64, slopes=_slopes(4), documents=_packed(rng, 2, 190, 3), causal=False, scale=0.02)
    _check(dtype, 2, 4, 2, n, 190, 64, cap=5.0, causal=False, scale=-0.1)
    _check(dtype, 2, 4, 2, n, 190, 64, causal=False, scale=0.0)
    _check(dtype, 1, 4, 2, n, n, 128, cap=1e4)       # hardly a cap at all
    _check(dtype, 1, 4, 2, n, n, 128, cap=512.0)
    _check(dtype, 1, 4, 2, n, n, 64, cap=1e20, scale=0.02)
    _check(dtype, 1, 4, 2, n, n, 128, cap=0.01)      # hardly a score left
    _check(dtype, 1, 4, 2, n, n, 128, cap=50.0, big=60.0)   # scores far beyond the cap


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("n", [2, 100, 400])
def test_documents_in_any_order_padding_and_empty_rows(rt, dtype, d, n):
    rng = np.random.default_rng(12)
    t = n + 37
    ids = rng.integers(0, 5, (2, t)).astype(np.int32)      # interleaved
    ids[0, t // 2 :] = -1                                    # padding: nobody sees it, it sees nobody
    ids[1, -1] = 77                                          # a document whose only token is the last one
    q, k, v = _rows(rng, (2, 4, n, d), dtype), _rows(rng, (2, 2, t, d), dtype), _rows(rng, (2, 2, t, d), dtype)
    want = scored(q, k, v, documents=ids, cap=10.0)
    k[0, :, t // 2 :], v[0, :, t // 2 :] = np.nan, np.inf    # ... whatever it holds
    got = ta.ScoredSdpa(softcap=10.0).eval(q, k, v, documents=ids).to_numpy()
    assert_within(got, *want)
    empty = ids[0, t - n :] < 0
    assert not got[0][:, empty].any()
    assert np.array_equal(got[1, :, -1], np.repeat(v[1, :, -1], 2, axis=0))
    all_padding = np.full((2, t), -3, np.int32)
    assert not ta.ScoredSdpa().eval(q, k, v, documents=all_padding).to_numpy().any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,n,t", [(64, 600, 600), (128, 300, 900)])
def test_packed_documents_with_a_tail_of_padding(rt, dtype, d, n, t):
    """Rows of padding beside rows of a document whose keys fill whole tiles: the ones see nothing, the others all of it."""
    ids = np.repeat(np.arange(6, dtype=np.int32), t // 6)[None].repeat(2, axis=0)
    ids[0, t - 77 :] = -1
    ids[1, 50:90] = -7
    got = _check(dtype, 2, 6, 2, n, t, d, documents=ids, slopes=_slopes(6))
    assert not got[0, :, n - 77 :].any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_fewer_keys_than_queries(rt, dtype):
    """Rows before the first key see nothing; a prefix shows them what it holds."""
    got = _check(dtype, 1, 4, 2, 50, 20, 64, cap=9.0)
    assert not got[:, :, :30].any()
    _check(dtype, 2, 4, 2, 50, 20, 64, prefix_lens=np.array([3, 900], np.int32))
    _check(dtype, 1, 4, 2, 200, 64, 128, slopes=_slopes(4))
    q = np.ones((1, 2, 3, 64), dtype)
    none = np.zeros((1, 1, 0, 64), dtype)
    assert not ta.ScoredSdpa(softcap=1.0).eval(q, none, none).to_numpy().any()


@pytest.mark.parametrize("dtype,b,hq,hkv,d", [(F16, 2, 8, 2, 128), (F32, 1, 4, 2, 64), (F16, 1, 14, 2, 64)])
def test_session_over_caches(rt, dtype, b, hq, hkv, d):
    """A prompt, a chunk, single tokens: over the caches as over the tensors they hold; the plain call where no rule is given."""
    rng = np.random.default_rng(13)
    kc, vc = ta.InPlaceKvCache(2), ta.InPlaceKvCache(2)
    whole_k, whole_v = (np.zeros((b, hkv, 0, d), dtype) for _ in range(2))
    op = ta.ScoredSdpa(softcap=25.0)
    slopes = _slopes(hq)
    for n in (130, 40, 1, 1, 5, 1):
        q = _rows(rng, (b, hq, n, d), dtype, 3.0)
        kn, vn = (_rows(rng, (b, hkv, n, d), dtype) for _ in range(2))
        kc.push(kn), vc.push(vn)
        whole_k, whole_v = np.concatenate([whole_k, kn], axis=2), np.concatenate([whole_v, vn], axis=2)
        dq = ta.DeviceTensor.from_numpy(q)
        got = op.eval_cached(dq, kc, vc, slopes=slopes).to_numpy()
        assert_within(got, *scored(q, whole_k, whole_v, cap=25.0, slopes=slopes))
        plain = ta.ScoredSdpa().eval_cached(dq, kc, vc).to_numpy()
        assert_within(plain, *scored(q, whole_k, whole_v))


def test_calls_queued_behind_each_other_and_refusals(rt):
    rng = np.random.default_rng(14)
    q, k, v = _rows(rng, (1, 8, 1, 128), F16, 4.0), _rows(rng, (1, 2, 4000, 128), F16), _rows(rng, (1, 2, 4000, 128), F16)
    dq, dk, dv = (ta.DeviceTensor.from_numpy(t) for t in (q, k, v))
    stream, op = ta.Stream(), ta.ScoredSdpa(softcap=20.0)
    outs = [op.eval(dq, dk, dv, stream=stream) for _ in range(20)]   # one workspace, one stream
    first = outs[0].to_numpy(stream)
    assert_within(first, *scored(q, k, v, cap=20.0))
    assert all(o.to_numpy(stream).tobytes() == first.tobytes() for o in outs)
    with pytest.raises(ta.TractRocmError, match="softcap"):
        ta.ScoredSdpa(softcap=-1.0).eval(dq, dk, dv)
    with pytest.raises(ta.TractRocmError, match="softcap"):
        ta.ScoredSdpa(softcap=float("nan")).eval(dq, dk, dv)
    with pytest.raises(ta.TractRocmError, match="slopes"):
        op.eval(dq, dk, dv, slopes=np.zeros(4, F32))
    with pytest.raises(ta.TractRocmError, match="documents"):
        op.eval(dq, dk, dv, documents=np.zeros((1, 3999), np.int32))
    with pytest.raises(ta.TractRocmError, match="out overlaps"):
        op.eval(dq, dk, dv, out=dq)
    with pytest.raises(ta.TractRocmError, match="documents need"):
        op.eval(np.zeros((1, 2, 4, 64), F16), np.zeros((1, 2, 3, 64), F16), np.zeros((1, 2, 3, 64), F16), documents=np.zeros((1, 3), np.int32))
    ring = [ta.WindowKvCache(2, 8) for _ in range(2)]
    quant = [ta.InPlaceKvCache(2, ta.Q8_0) for _ in range(2)]
    for c in ring + quant:
        c.push(_rows(rng, (1, 2, 4, 128), F16))
    with pytest.raises(ta.TractRocmError, match="in order"):
        op.eval_cached(dq, *ring)
    with pytest.raises(ta.TractRocmError, match="block-quantised"):
        op.eval_cached(dq, *quant)
