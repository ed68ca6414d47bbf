"""RMS norm of query and key heads with the rotation in one pass, and the whole step with it, against 64 bits."""
import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, norm_rope
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


def _angles(rng, batch, n, d, dtype):
    a = (rng.integers(0, 30000, (batch, 1, 1, 1)) + np.arange(n)[None, None, :, None]) * 10000.0 ** (-np.arange(0, d, 2) / d)
    a = np.concatenate([a, a], axis=-1)
    return np.cos(a).astype(dtype), np.sin(a).astype(dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,hq,hkv,n,d,cs_batch", [
    (1, 32, 8, 1, 128, 1), (3, 14, 2, 5, 64, 3), (2, 5, 5, 33, 256, 2), (1, 40, 8, 700, 128, 1), (64, 4, 1, 1, 64, 64),
    (2, 3, 1, 7, 96, 1),       # a head size without a kernel of its own
    (1, 2, 2, 3, 2, 1), (2, 7, 3, 2, 1030, 2), (1, 64, 8, 600, 64, 1), (5, 0, 3, 2, 64, 1), (5, 3, 0, 2, 64, 5)])
def test_norm_rope(rt, dtype, batch, hq, hkv, n, d, cs_batch):
    rng = np.random.default_rng(1)
    q, k = _rows(rng, (batch, hq, n, d), dtype, 3.0), _rows(rng, (batch, hkv, n, d), dtype, 0.2)
    wq, wk = (rng.uniform(0.5, 1.5, d).astype(dtype) for _ in range(2))
    cos, sin = _angles(rng, cs_batch, n, d, dtype)
    got_q, got_k = ta.QkNormRope(1e-5).eval(q, k, wq, wk, cos, sin)
    for got, x, w in ((got_q, q, wq), (got_k, k, wk)):
        if x.size:
            assert_within(got.to_numpy(), *norm_rope(x, w, cos, sin, 1e-5))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shift", [0, 1])   # 1: a base that no 16-byte access fits
@pytest.mark.parametrize("batch,hq,hkv,n,d", [(2, 6, 2, 37, 64), (1, 32, 8, 300, 128), (4, 3, 1, 1, 128)])
def test_views_of_fused_rows(rt, dtype, shift, batch, hq, hkv, n, d):
    rng = np.random.default_rng(2)
    width = (hq + 2 * hkv) * d
    flat = _rows(rng, (shift + batch * n * width,), dtype)
    rows = flat[shift:].reshape(batch, n, hq + 2 * hkv, d)
    dev = ta.DeviceTensor.from_numpy(flat)
    es = np.dtype(dtype).itemsize
    cos, sin = _angles(rng, batch, n, d, dtype)
    st = (n * width, d, width, 1)
    q = ta.DeviceTensor((batch, hq, n, d), dtype, ptr=dev.ptr.value + shift * es, owner=dev)
    k = ta.DeviceTensor((batch, hkv, n, d), dtype, ptr=dev.ptr.value + (shift + hq * d) * es, owner=dev)
    c, s = (ta.DeviceTensor.from_numpy(t) for t in (cos, sin))
    got = ta.QkNormRope(1e-6).eval(q, k, None, None, c, s, q_strides=st, k_strides=st)
    for g, x in zip(got, (rows[:, :, :hq], rows[:, :, hq : hq + hkv])):
        assert_within(g.to_numpy(), *norm_rope(np.ascontiguousarray(x.transpose(0, 2, 1, 3)), None, cos, sin, 1e-6))
    assert dev.to_numpy().tobytes() == flat.tobytes()


@pytest.mark.parametrize("dtype,d", [(F16, 128), (F32, 64), (F16, 24)])
def test_in_place_rows_of_zeros_and_large_values(rt, dtype, d):
    rng = np.random.default_rng(3)
    q, k = _rows(rng, (2, 5, 9, d), dtype), _rows(rng, (2, 2, 9, d), dtype)
    q[0, 1, 3] = 0.0
    q[1, 2, 4] *= dtype(3e3 if dtype == F16 else 1e15)
    cos, sin = _angles(rng, 1, 9, d, dtype)
    dq, dk, c, s = (ta.DeviceTensor.from_numpy(t) for t in (q, k, cos, sin))
    ta.QkNormRope(1e-6).eval(dq, dk, None, None, c, s, q_out=dq, k_out=dk)
    assert_within(dq.to_numpy(), *norm_rope(q, None, cos, sin, 1e-6))
    assert_within(dk.to_numpy(), *norm_rope(k, None, cos, sin, 1e-6))
    assert not dq.to_numpy()[0, 1, 3].any()


def test_nan_stays_in_its_row(rt):
    rng = np.random.default_rng(4)
    q, k = _rows(rng, (1, 4, 6, 64), F16), _rows(rng, (1, 1, 6, 64), F16)
    q[0, 2, 1, 5], k[0, 0, 3, 0] = np.nan, np.inf
    cos, sin = _angles(rng, 1, 6, 64, F16)
    got_q, got_k = (t.to_numpy() for t in ta.QkNormRope().eval(q, k, None, None, cos, sin))
    bad_q, bad_k = np.isnan(got_q).all(axis=-1), np.isnan(got_k).any(axis=-1)
    assert bad_q[0, 2, 1] and bad_q.sum() == 1 and bad_k[0, 0, 3] and bad_k.sum() == 1
    assert np.isfinite(got_q[~bad_q]).all() and np.isfinite(got_k[~bad_k]).all()


def test_strides_are_read_at_every_call(rt):
    rng = np.random.default_rng(20)
    rows = rng.standard_normal((3, 8, 64), dtype=np.float32)
    cos, sin = (ta.DeviceTensor.from_numpy(rng.standard_normal((1, 1, 3, 64), dtype=np.float32)) for _ in range(2))
    x, strides, op = ta.DeviceTensor.from_numpy(rows), [3 * 8 * 64, 64, 8 * 64, 1], ta.QkNormRope(1e-6)
    q, k = (ta.DeviceTensor((1, 4, 3, 64), np.float32, ptr=x.ptr, owner=x) for _ in range(2))
    want = norm_rope(np.ascontiguousarray(rows[:, :4].transpose(1, 0, 2))[None], None, cos.to_numpy(), sin.to_numpy(), 1e-6)
    assert_within(op.eval(q, k, None, None, cos, sin, q_strides=strides)[0].to_numpy(), *want)
    strides[:] = [4 * 3 * 64, 3 * 64, 64, 1]     # the same list: now the buffer's first rows as they lie
    want = norm_rope(rows.reshape(-1, 64)[:12].reshape(1, 4, 3, 64), None, cos.to_numpy(), sin.to_numpy(), 1e-6)
    assert_within(op.eval(q, k, None, None, cos, sin, q_strides=strides)[0].to_numpy(), *want)


def test_stream_and_refusals(rt):
    rng = np.random.default_rng(5)
    q, k = _rows(rng, (1, 4, 3, 64), F16), _rows(rng, (1, 2, 3, 64), F16)
    cos, sin = _angles(rng, 1, 3, 64, F16)
    dq, dk, c, s = (ta.DeviceTensor.from_numpy(t) for t in (q, k, cos, sin))
    stream = ta.Stream()
    got, _ = ta.QkNormRope().eval(dq, dk, None, None, c, s, stream=stream)
    assert_within(got.to_numpy(stream), *norm_rope(q, None, cos, sin, 1e-6))
    op = ta.QkNormRope()
    with pytest.raises(ta.TractRocmError, match="overlap"):
        op.eval(dq, dk, None, None, c, s, q_out=ta.DeviceTensor(q.shape, F16, ptr=dq.ptr.value + 128, owner=dq))
    with pytest.raises(ta.TractRocmError, match="overlap"):
        op.eval(dq, dk, None, None, c, s, q_out=dq, q_strides=(768, 64, 256, 1))
    with pytest.raises(ta.TractRocmError, match="datum type"):
        op.eval(dq, ta.DeviceTensor(k.shape, F32), None, None, c, s)
    with pytest.raises(ta.TractRocmError, match="weight"):
        op.eval(dq, dk, ta.DeviceTensor((32,), F16), None, c, s)


@pytest.mark.parametrize("fmt", [None, ta.Q8_0])
@pytest.mark.parametrize("batch,hq,hkv,d,chunks,fused", [(2, 8, 2, 128, (40, 1, 1, 3), True), (1, 4, 4, 128, (1, 1, 70), False), (3, 6, 1, 128, (5, 1), True)])
def test_step_equals_its_parts(rt, fmt, batch, hq, hkv, d, chunks, fused):
    """eval_norm_rope_into = QkNormRope, then eval_into: the same bytes in the caches and the same output."""
    rng = np.random.default_rng(6)
    wq, wk = (ta.DeviceTensor.from_numpy(rng.uniform(0.5, 1.5, d).astype(F16)) for _ in range(2))
    whole, parts = (ta.InPlaceKvSdpa(axis=2, causal=True, storage_format=fmt).state() for _ in range(2))
    for n in chunks:
        width = hq + 2 * hkv
        rows = _rows(rng, (batch, n, width, d), F16)
        dev = ta.DeviceTensor.from_numpy(rows)
        q, k, v = (np.ascontiguousarray(rows[:, :, a:b].transpose(0, 2, 1, 3)) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, width)))
        cos, sin = (ta.DeviceTensor.from_numpy(t) for t in _angles(rng, 1, n, d, F16))
        if fused:
            st = (n * width * d, d, width * d, 1)
            views = [ta.DeviceTensor((batch, h, n, d), F16, ptr=dev.ptr.value + off * d * 2, owner=dev) for h, off in ((hq, 0), (hkv, hq), (hkv, hq + hkv))]
            out = whole.eval_norm_rope_into(*views, wq, wk, 1e-6, cos, sin, q_strides=st, k_strides=st, v_strides=st)
        else:
            out = whole.eval_norm_rope_into(*(ta.DeviceTensor.from_numpy(t) for t in (q, k, v)), wq, wk, 1e-6, cos, sin)
        nq, nk = ta.QkNormRope(1e-6).eval(ta.DeviceTensor.from_numpy(q), ta.DeviceTensor.from_numpy(k), wq, wk, cos, sin)
        if fused:
            parts.k.push(nk), parts.v.push(ta.DeviceTensor.from_numpy(v))
            want = parts.attend(nq)
        else:
            want = parts.eval_into(nq, nk, ta.DeviceTensor.from_numpy(v))
        assert out.to_numpy().tobytes() == want.to_numpy().tobytes()
        assert whole.k.valid_contiguous().tobytes() == parts.k.valid_contiguous().tobytes()
        assert whole.v.valid_contiguous().tobytes() == parts.v.valid_contiguous().tobytes()
    n = whole.k.len()
    with pytest.raises(ta.TractRocmError, match="datum type"):
        whole.eval_norm_rope_into(nq, nk, nk, ta.DeviceTensor((d,), F32), None, 1e-6, cos, sin)
    with pytest.raises(ta.TractRocmError):
        whole.eval_norm_rope_into(nq, nk, nk, None, None, -1.0, cos, sin)
    assert whole.k.len() == n and whole.v.len() == n
