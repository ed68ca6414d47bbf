"""Beam search's choice against 64 bits: tokens and parents equal, scores within a half step of f32 and the sums' own errors."""
import numpy as np
import pytest

import tract_amd as ta
from tests import paged_ref as ref
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy


def _check(logits, scores, keep, ended=None, eos=-1, row_stride=0, device_logits=None):
    want = ref.select(logits, scores, keep, ended, eos)
    got = ta.BeamSelect(keep, eos).eval(up(logits) if device_logits is None else device_logits, up(scores), ended=None if ended is None else up(ended), row_stride=row_stride)
    got = {name: t.to_numpy() for name, t in got.items()}
    w, g = want["scores"], got["scores"].astype(np.float64)
    sure = np.isfinite(w)
    assert (g[~sure] == w[~sure]).all()
    # A weight exp(x - max) is off by the half steps (2^-24) of the difference and of its product with log2 e, each on the exponent d, and by
    # the exponential's two; seven f32 additions of a piece follow, the rest is f64.  Weighted by the weights themselves d is at most ln(vocab)
    # on average (its entropy is d + ln(sum), and the sum is at least 1): 2 * 21.5 + 2 + 7 of a vocabulary below 2^31, so the sum and its
    # logarithm are within 64 half steps.  Then the rounding to f32.
    off = 64 * 2.0 ** -24
    assert (np.abs(g[sure] - w[sure]) <= 2.0 ** -24 * np.abs(w[sure]) + off).all(), np.abs(g[sure] - w[sure]).max()
    for name in ("parents", "tokens", "ended"):
        np.testing.assert_array_equal(got[name], want[name], err_msg=name)
    return got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 4, 1, 4), (3, 2, 5, 4), (2, 3, 7, 21), (1, 1, 64, 64), (2, 4, 100, 8), (5, 8, 1000, 16), (1, 4, 2047, 4), (1, 4, 2048, 4), (1, 4, 2049, 4), (2, 64, 77, 64), (1, 2, 8191, 3),
    (1, 2, 8193, 5), (2, 5, 32001, 10), (70, 4, 8200, 8), (40, 8, 4001, 16), (1, 64, 20000, 64), (300, 1, 300, 2)])
def test_select(rt, dtype, batch, beams, vocab, keep):
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((batch, beams, vocab)) * 4).astype(dtype)
    _check(logits, (-rng.random((batch, beams)) * 10).astype(F32), keep)
    _check(logits, np.zeros((batch, beams), F32), keep, eos=vocab // 2)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("vocab", [9, 3000, 20001])
@pytest.mark.parametrize("keep", [1, 7, 64])
def test_equal_values_go_to_the_lowest(rt, dtype, vocab, keep):
    """Beams that are copies of one another, rows of one value, of two, and of whole numbers."""
    rng = np.random.default_rng(keep)
    b, w = 3, 8
    keep = min(keep, w * vocab)
    same = np.repeat(rng.standard_normal((b, 1, vocab)), w, axis=1).astype(dtype)
    zero = np.zeros((b, w), F32)
    _check(same, zero, keep)
    _check(np.full((b, w, vocab), 1.5, dtype), zero, keep)
    _check(rng.integers(0, 2, (b, w, vocab)).astype(dtype), zero, keep)
    _check(np.repeat(rng.integers(-3, 3, (b, 1, vocab)), w, axis=1).astype(dtype), zero, keep)
    signs = np.zeros((b, w, vocab), dtype)
    signs[..., ::2] = -0.0                                    # both zeros are one number
    _check(signs, zero, keep)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_sorted_rows_and_clustered_peaks(rt, dtype):
    """The largest values side by side: more of them in a lane or a wave than it has on average."""
    n = 9000
    up_hill = np.linspace(-4, 4, n)
    steps = np.stack([up_hill, up_hill[::-1], np.where(np.arange(n) % 4096 < 64, 5 + np.arange(n) / n, 0.0), np.where(np.arange(n) < 300, np.arange(n) / 64 + 1, -2.0)])
    logits = np.stack([steps, steps[::-1]]).astype(dtype)
    for keep in (1, 16, 64):
        _check(logits, np.array([[0, -0.25, -0.5, -0.75]] * 2, F32), keep)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_masked_and_infinite_values(rt, dtype):
    rng = np.random.default_rng(2)
    b, w, n, keep = 4, 4, 5000, 8
    logits = rng.standard_normal((b, w, n)).astype(dtype)
    logits[0, :, 10:] = -np.inf                    # fewer finite continuations than are kept
    logits[0, :, 12] = np.nan
    logits[1, 0] = -np.inf                         # a row that leaves nothing
    logits[1, 1] = np.nan
    logits[1, 2, 77] = np.inf
    logits[2] = -np.inf                            # a request that leaves nothing
    logits[3, :, 1:] = np.finfo(dtype).min
    logits[3, :, 3:] = np.nan
    scores = (-rng.random((b, w))).astype(F32)
    _check(logits, scores, keep)
    for keep in (1, 40, 64):
        _check(logits, scores, keep, eos=3)
    scores[0, 1:] = -np.inf                        # the first step of a search
    scores[1, 3], scores[3, 0], scores[3, 1] = np.nan, np.inf, -np.inf
    _check(logits, scores, keep)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_ended_beams(rt, dtype):
    rng = np.random.default_rng(3)
    for vocab, eos in ((3000, 2), (20, 19), (40, 0), (20001, 20000)):
        logits = (rng.standard_normal((6, 4, vocab)) * 2).astype(dtype)
        scores = (-rng.random((6, 4)) * 3).astype(F32)
        ended = (rng.random((6, 4)) < 0.5).astype(I32) * 7
        ended[0], ended[1] = 0, 1
        logits[2, :, 3:] = -np.inf
        scores[1, 2], scores[1, 3] = -np.inf, np.nan
        for keep in (1, 4, 8, 64):
            if keep <= 4 * vocab:
                got = _check(logits, scores, keep, ended, eos)
                assert (got["tokens"][1, :min(keep, 2)] == eos).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_of_a_wider_tensor_and_odd_places(rt, dtype):
    rng = np.random.default_rng(4)
    b, w, vocab = 2, 3, 4099
    for stride, offset in ((4099, 0), (4100, 1), (5001, 3), (4112, 8)):
        base = (rng.standard_normal(offset + b * w * stride) * 3).astype(dtype)
        logits = np.lib.stride_tricks.as_strided(base[offset:], (b, w, vocab), tuple(x * base.itemsize for x in (w * stride, stride, 1))).copy()
        d = up(base)
        view = ta.DeviceTensor((b, w, vocab), dtype, ptr=d.ptr.value + offset * base.itemsize, owner=d)
        _check(logits, (-rng.random((b, w))).astype(F32), 6, row_stride=stride, device_logits=view)


def test_large_scores_and_peaked_rows(rt):
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((2, 4, 6000)) * 30).astype(F32)
    logits[0, 0, 5] = 1000.0
    logits[1, :, 100] = -3e38
    _check(logits, np.array([[-1000.0, -2000.5, -1e5, -990.0], [-1e-3, -1e-6, -500.0, -1.0]], F32), 8)


def test_shapes_and_types_are_refused(rt):
    x, s = up(np.zeros((2, 3, 50), F16)), up(np.zeros((2, 3), F32))
    for bad in ((up(np.zeros((6, 50), F16)), s), (x, up(np.zeros((2, 3), F16))), (x, up(np.zeros((2, 2), F32))), (up(np.zeros((2, 3, 50), I32)), s)):
        with pytest.raises(ta.TractRocmError):
            ta.BeamSelect(2).eval(*bad)
    with pytest.raises(ta.TractRocmError):
        ta.BeamSelect(2, eos=1).eval(x, s, ended=up(np.zeros((2, 3), F32)))
    with pytest.raises(ta.TractRocmError):
        ta.BeamSelect(2).eval(x, s, ended=up(np.zeros((2, 3), I32)))
    with pytest.raises(ta.TractRocmError):
        ta.BeamSelect(2).eval(x, s, out={"scores": up(np.zeros((2, 3), F32))})
    with pytest.raises(ta.TractRocmError):
        ta.BeamSelect(200).eval(x, s)


def test_more_requests_than_a_launch_counts(rt):
    """16384 requests have a counter each in a launch; parents of the ones behind them are rows of the whole batch."""
    rng = np.random.default_rng(6)
    logits = (rng.standard_normal((16400, 2, 9)) * 2).astype(F32)
    got = _check(logits, (-rng.random((16400, 2))).astype(F32), 3)
    assert got["parents"].max() >= 2 * 16399


def test_keep_that_changes_from_call_to_call(rt):
    rng = np.random.default_rng(7)
    logits, scores = (rng.standard_normal((2, 3, 500))).astype(F16), (-rng.random((2, 3))).astype(F32)
    op = ta.BeamSelect(2)
    for keep in (2, 60, 5):
        op.keep = keep
        got, want = op.eval(up(logits), up(scores)), ref.select(logits, scores, keep)
        for name in ("parents", "tokens"):
            np.testing.assert_array_equal(got[name].to_numpy(), want[name])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("batch,beams,vocab,keep", [(1, 8, 40000, 16), (1, 2, 128256, 64), (2, 64, 9000, 64), (1, 40, 16385, 3), (3, 8, 50257, 16)])
def test_more_candidates_than_a_workgroup_holds(rt, dtype, batch, beams, vocab, keep):
    """Parts of a request whose candidates are looked at by their best ones first: scores alike, far apart (one beam has all of the choice), of beams
    that have ended or are gone, and rows sorted both ways, equal throughout or with few numbers."""
    rng = np.random.default_rng(vocab + keep)
    logits = (rng.standard_normal((batch, beams, vocab)) * 3).astype(dtype)
    near, far = (-rng.random((batch, beams))).astype(F32), (-200.0 * rng.random((batch, beams))).astype(F32)
    _check(logits, near, keep)
    _check(logits, far, keep)
    ended = (rng.random((batch, beams)) < 0.5).astype(I32)
    gone = near.copy()
    gone[:, 1] = -np.inf
    _check(logits, gone, keep, ended, vocab - 1)
    _check(np.sort(logits, axis=-1), near, keep)
    _check(-np.sort(logits, axis=-1), far, keep)
    _check(np.zeros_like(logits), near, keep)
    _check(np.zeros_like(logits), np.zeros_like(near), keep)
    few = np.full_like(logits, -np.inf)
    few[..., ::vocab // 3] = logits[..., ::vocab // 3]
    _check(few, near, keep)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_behind_four_gibibytes(rt, dtype):
    """Rows 2^29 elements apart, of which nine hold logits: put there as rows of pages, whose strides say where."""
    rng, b, w, vocab, apart = np.random.default_rng(13), 3, 3, 5003, 1 << 29
    logits = (rng.standard_normal((b, w, vocab)) * 3).astype(dtype)
    rows, size = up(logits.reshape(b * w, 1, vocab)), (b * w - 1) * apart + vocab
    far, other = ta.DeviceTensor((size,), dtype), ta.DeviceTensor((size,), dtype)
    pages = lambda t: ta.DeviceTensor((b * w, 1, 1, vocab), dtype, ptr=t.ptr.value, owner=t)  # noqa: E731
    ta.PagedAppend().eval(rows, rows, up(np.arange(b * w, dtype=I32)), pages(far), pages(other), page_strides=(apart, vocab, vocab))
    view = ta.DeviceTensor((b, w, vocab), dtype, ptr=far.ptr.value, owner=far)
    _check(logits, (-rng.random((b, w))).astype(F32), 6, row_stride=apart, device_logits=view)


def test_arrays_of_the_host_are_taken_too(rt):
    rng = np.random.default_rng(8)
    logits, scores = rng.standard_normal((2, 3, 300)).astype(F32), (-rng.random((2, 3))).astype(F32)
    want = ref.select(logits, scores, 4)
    for x, s in ((logits, scores), (up(logits), scores), (logits, up(scores))):
        got = ta.BeamSelect(4).eval(x, s)
        for name in ("parents", "tokens"):
            np.testing.assert_array_equal(got[name].to_numpy(), want[name])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("vocab", [2, 3, 17, 3000])
def test_rows_that_are_others_shifted_tie(rt, dtype, vocab):
    """Logits of one beam plus a whole number are the same continuation probabilities: equal values, to the lowest beam."""
    rng = np.random.default_rng(vocab)
    base, by = rng.integers(-4, 5, (5, 1, vocab)), rng.integers(-9, 10, (5, 6, 1))
    keep = min(12, 6 * vocab)
    _check((base + by).astype(dtype), np.zeros((5, 6), F32), keep)
    _check((rng.permuted(np.repeat(base, 6, axis=1), axis=2) + by).astype(dtype), np.full((5, 6), -3.25, F32), keep)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_sums_that_differ_in_the_last_places(rt, dtype):
    """Beams that differ in one logit of 28 to 33 below the largest: their sums, in parts of 7e-13 to 5e-15, and what is chosen with them, in an order
    that is not that of the beams.  (The terms that the rows share are off by the same; 5e-15 is 20 steps of 64 bits.)"""
    rng = np.random.default_rng(11)
    row = (-12 + rng.standard_normal(20001)).astype(dtype)
    logits = np.repeat(row[None, None], 6, axis=1).repeat(2, axis=0)
    logits[..., 777] = 0
    logits[0, :, 5000] = -28 - np.arange(6)
    logits[1, :, 19999] = -28 - np.array([2, 0, 5, 1, 4, 3])
    got = _check(logits, np.zeros((2, 6), F32), 12)
    assert got["parents"][0, :6].tolist() == [5, 4, 3, 2, 1, 0] and (got["parents"][1, :6] - 6).tolist() == [2, 4, 5, 0, 3, 1]
