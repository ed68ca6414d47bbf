"""Beam search's choice over masked vocabularies: rows whose values are finite and far from zero, and sums made again over rows with -inf."""
import numpy as np
import pytest

import tract_amd as ta
from tests import paged_ref as ref
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy
MASKS = [-1e9, -1e10, -1e12, -1e15, -1e18, -1e25, -1e30, -1e38, float(np.finfo(F32).min)]


def _check(logits, scores, keep, ended=None, eos=-1):
    """The choice into buffers that hold something else; the bound on scores as tests/test_gpu_beam_select.py derives it, with a weight's exponent off by
    three half steps of itself: 3 * 21.5 + 2 + 7 half steps of the sum, and the score's own."""
    want = ref.select(logits, scores, keep, ended, eos)
    shape = (logits.shape[0], keep)
    out = {"scores": up(np.full(shape, 77.0, F32)), **{name: up(np.full(shape, -777, I32)) for name in ("parents", "tokens", "ended")}}
    got = ta.BeamSelect(keep, eos).eval(up(logits), up(scores), ended=None if ended is None else up(ended), out=out)
    got = {name: t.to_numpy() for name, t in got.items()}
    w, g = want["scores"], got["scores"].astype(np.float64)
    for name in ("parents", "tokens", "ended"):
        np.testing.assert_array_equal(got[name], want[name], err_msg=name)
    sure = np.abs(w) < float(np.finfo(F32).max) + 2.0 ** 103     # (f32 rounds others to infinities: its last step, halved, is 2^103)
    assert np.isneginf(g[~sure]).all()
    assert (np.abs(g[sure] - w[sure]) <= 2.0 ** -24 * np.abs(w[sure]) + 74 * 2.0 ** -24).all(), np.abs(g[sure] - w[sure]).max()
    return got


def _masked(rng, beams, vocab, mask, allowed):
    """`allowed` tokens of every beam have a logit, the others the mask."""
    logits = np.full((2, beams, vocab), mask, F32)
    for i in range(2):
        for b in range(beams):
            at = rng.choice(vocab, allowed, replace=False)
            logits[i, b, at] = rng.standard_normal(allowed) * 3
    return logits


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("vocab", [70, 3001, 40000])
def test_few_tokens_are_allowed(rt, mask, vocab):
    """All that most waves see is the mask."""
    rng = np.random.default_rng(vocab)
    for beams, allowed, keep in ((1, 20, 4), (4, 20, 8), (4, 3, 12), (4, 1, 4)):
        _check(_masked(rng, beams, vocab, mask, allowed), (-rng.random((2, beams))).astype(F32), keep)


@pytest.mark.parametrize("value", MASKS + [1e10, 1e20, 3e38])
@pytest.mark.parametrize("vocab", [9, 3001, 40000])
def test_rows_of_one_far_value(rt, value, vocab):
    """A row that is the mask throughout leaves every token score - log(vocab): alone, in all beams, and beside ordinary beams that it wins and loses against."""
    rng, keep = np.random.default_rng(3), 6
    row = np.full(vocab, value, F32)
    _check(row[None, None], np.array([[-1.5]], F32), keep)
    _check(np.tile(row, (2, 4, 1)), (-rng.random((2, 4))).astype(F32), keep)
    _check(np.tile(row, (1, 4, 1)), np.zeros((1, 4), F32), keep)
    mixed = (rng.standard_normal((3, 4, vocab)) * 3).astype(F32)
    mixed[0, 2], mixed[1, 0], mixed[2, 1:3] = row, row, row
    for lead in (0.0, 8.0, 30.0):
        scores = (-rng.random((3, 4))).astype(F32)
        scores[0, 2] += lead
        scores[1, 0] += lead
        scores[2, 1:3] += lead
        _check(mixed, scores, keep)


@pytest.mark.parametrize("far", [1e6, 1e8, 1e10, 1e30, 3e38])
def test_a_largest_value_far_above(rt, far):
    """One token has nearly all of the weight, and what is below it is far away, too."""
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((2, 3, 9000)) * 3).astype(F32)
    logits[0, :, 4321] = far
    logits[1, 1, [7, 8999]] = far
    _check(logits, np.array([[-1.0, -2.0, -3.0], [-0.5, -0.25, -0.75]], F32), 7)


@pytest.mark.parametrize("by", [2.0 ** 20, 2.0 ** 23])
def test_rows_far_from_zero(rt, by):
    """Ordinary differences around a value whose last place is 2^-3 or 1: the sum is as good as that of rows around zero."""
    rng = np.random.default_rng(6)
    logits = (rng.integers(-12, 1, (2, 4, 20001)) + by).astype(F32)
    logits[:, :, 777] = by + np.array([3, 4, 5, 6])
    _check(logits, (-rng.random((2, 4))).astype(F32), 4)
    _check(-logits, (-rng.random((2, 4))).astype(F32), 4)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("vocab", [13, 3001, 40000])
def test_sums_made_again_over_masked_rows(rt, dtype, vocab):
    """Beams that are copies of one another, or others shifted, whose vocabulary is mostly masked: values so near that the exact sums decide, over terms of
    -inf, of the type's lowest value and NaN."""
    rng = np.random.default_rng(vocab)
    base = rng.integers(-4, 5, (3, 1, vocab)).astype(dtype)
    for mask in (-np.inf, np.finfo(dtype).min, np.nan):
        hidden = rng.random(base.shape) < 0.7
        hidden[..., 5] = False
        same = np.where(hidden, dtype(mask), base).repeat(5, axis=1)
        zero = np.zeros((3, 5), F32)
        _check(same, zero, 11)
        _check(np.where(hidden, dtype(mask), base + rng.integers(-9, 10, (3, 5, 1)).astype(dtype)), zero, 11)
        _check(rng.permuted(same, axis=2), zero - 3.25, 11)


@pytest.mark.parametrize("vocab", [7, 3001, 40000])
@pytest.mark.parametrize("keep", [1, 5, 64])
def test_logits_that_one_value_stands_for(rt, vocab, keep):
    """Where 64 bits hold the same score + log softmax for logits that differ, the lowest places are chosen, not the largest logits: logits next to nothing
    (alone, among others, beside a far one), and scores that take all of them in."""
    rng = np.random.default_rng(vocab + keep)
    keep = min(keep, 3 * vocab)
    score = np.zeros((2, 3), F32)
    tiny = (rng.standard_normal((2, 3, vocab)) * 1e-20).astype(F32)
    _check(tiny, score, keep)
    _check(tiny, (-rng.random((2, 3))).astype(F32), keep)
    some = np.where(rng.random(tiny.shape) < 0.5, tiny, F32(-1)).astype(F32)
    some[:, :, vocab // 2] = [3, 2, 2]
    _check(some, score, keep)
    far = (rng.standard_normal((2, 3, vocab)) * 3).astype(F32)
    far[..., vocab // 3] = 1e25
    _check(far, score, keep)
    for dtype, large in ((F32, -1e17), (F32, 1e30), (F16, -3e16), (F16, 1e9)):
        logits = (rng.standard_normal((2, 3, vocab)) * (3 if abs(large) > 1e10 else 1e-7)).astype(dtype)
        _check(logits, np.full((2, 3), large, F32), keep)
        _check(logits, np.array([[large, large, 1.0], [large, -1.0, large]], F32), keep, np.array([[0, 1, 0], [1, 0, 0]], I32), vocab - 2)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_more_of_them_than_are_listed(rt, dtype):
    """Candidates of equal value beyond what the join lists: 64 beams of 64 candidates each in every part."""
    rng = np.random.default_rng(9)
    tiny = (rng.integers(-9, 10, (1, 64, 2500)) * (1e-20 if dtype == F32 else 6e-8)).astype(dtype)
    _check(tiny, np.full((1, 64), 0.0 if dtype == F32 else 1e9, F32), 64)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("score", [2.0 ** 51, 2.0 ** 52, 1e15, 3e12])
def test_values_that_their_own_rounding_decides(rt, dtype, score):
    """Scores whose last place is about the steps of the logits, which lie half way between two values of 64 bits as often as not: the least that a sum is
    off by turns them the other way, and with them equal ones and their order, in one beam and between beams that have the same score."""
    rng, vocab = np.random.default_rng(12), 10481
    logits = (rng.integers(-400, 401, (2, 5, vocab)) / 4).astype(dtype)
    logits[..., 5000] = 60000
    scores = np.full((2, 5), -score, F32)
    for keep in (1, 7, 50):
        _check(logits, scores, keep)
        _check(np.ascontiguousarray(logits[:, :1]), np.ascontiguousarray(scores[:, :1]), keep)
    scores[1, 1:4] *= F32(0.75)
    _check(logits, scores, 50)
