"""A query row of NaN comes out as NaN, and no other row does, however many parts its keys go in."""
import numpy as np
import pytest

import tract_amd as ta
from tests.attention_ref import assert_within, scored, shared
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def _rows(rng, shape, dtype, scale=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(dtype)


def _only(got, at, want, bound):
    """got[at] is NaN throughout, the rest is what it was to be."""
    assert np.isnan(got[at]).all(), got[at]
    got = got.copy()
    got[at] = want[at]
    assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,hq,hkv,p,sq,d", [
    ([3, 0, 40], 14, 2, 777, 1, 64), ([100, 31, 900], 8, 2, 2000, 1, 128),    # tiles of 16 rows, joined by the last to arrive
    ([9, 70] * 20, 32, 2, 4000, 1, 128), ([9, 70] * 20, 64, 2, 4000, 1, 64),  # f16: tiles of 128 rows over the prefix, joined by a launch
    ([40, 200], 32, 2, 300, 5, 128), ([5, 0], 8, 1, 700, 6, 64),              # several queries of a sequence
    ([5, 2, 300], 6, 3, 400, 1, 80), ([2, 600], 4, 2, 0, 2, 48)])             # head sizes without a kernel of their own
def test_shared_prefix(rt, dtype, lens, hq, hkv, p, sq, d):
    rng = np.random.default_rng(41)
    n, room = len(lens), max(lens)
    q, pk, pv = _rows(rng, (n, hq, sq, d), dtype, 2.0), _rows(rng, (1, hkv, max(p, 1), d), dtype), _rows(rng, (1, hkv, max(p, 1), d), dtype)
    k, v = (_rows(rng, (n, hkv, room, d), dtype) for _ in range(2))
    want = shared(q, pk[0, :, :p], pv[0, :, :p], [t[:, :i] for t, i in zip(k, lens)], [t[:, :i] for t, i in zip(v, lens)])
    at = n - 1, hq // 2, sq - 1
    q[at][d // 3] = np.nan
    op = ta.SharedPrefixSdpa()
    for _ in range(2):
        _only(op.eval(q, pk, pv, k, v, lens, prefix_len=p).to_numpy(), at, *want)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("b,hq,hkv,n,t,d", [
    (2, 8, 2, 1, 5000, 128), (1, 4, 1, 1, 9000, 64), (1, 32, 4, 1, 300, 128),    # single tokens, in parts and whole
    (1, 8, 2, 6, 5000, 128), (1, 4, 2, 40, 6000, 64), (1, 8, 2, 100, 130, 64),   # a few queries, a chunk, a prompt
    (1, 6, 2, 3, 700, 96), (2, 2, 1, 1, 40, 48)])                                # head sizes without a kernel of their own
@pytest.mark.parametrize("cap,documents", [(0.0, False), (20.0, False), (0.0, True)])
def test_scored(rt, dtype, b, hq, hkv, n, t, d, cap, documents):
    rng = np.random.default_rng(42)
    q, k, v = _rows(rng, (b, hq, n, d), dtype, 3.0), _rows(rng, (b, hkv, t, d), dtype), _rows(rng, (b, hkv, t, d), dtype)
    rules = dict(slopes=(2.0 ** -np.arange(hq)).astype(F32), documents=(np.arange(t) * 3 // t)[None].repeat(b, 0).astype(np.int32) if documents else None)
    want = scored(q, k, v, cap=cap, **rules)
    at = b - 1, hq - 1, n // 2
    q[at][0] = np.nan
    _only(ta.ScoredSdpa(softcap=cap).eval(q, k, v, **rules).to_numpy(), at, *want)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 48])
def test_a_row_that_sees_nothing_is_zeros_whatever_its_query_holds(rt, dtype, d):
    rng = np.random.default_rng(43)
    q, k, v = _rows(rng, (1, 4, 3, d), dtype), _rows(rng, (1, 2, 3000, d), dtype), _rows(rng, (1, 2, 3000, d), dtype)
    ids = np.zeros((1, 3000), np.int32)
    ids[0, -1] = -1
    want = scored(q, k, v, documents=ids)
    q[:, :, -1] = np.nan
    got = ta.ScoredSdpa().eval(q, k, v, documents=ids).to_numpy()
    assert not got[:, :, -1].any()
    assert_within(got, *want)
    empty = np.zeros((1, 2, 0, d), dtype)
    assert not ta.ScoredSdpa().eval(q, empty, empty).to_numpy().any()
