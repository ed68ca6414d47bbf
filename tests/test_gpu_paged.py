"""Tables, appends, reordering and attention over pages against plain restatements (tests/paged_ref.py)."""
import ctypes as C

import numpy as np
import pytest

import tract_amd as ta
from tests import paged_ref as ref
from tests.attention_ref import assert_within
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy


def ints(x):
    return up(np.asarray(x, I32))


# ---- plan --------------------------------------------------------------------------------------------------


def _tables(rng, lens, page, width, n_pages):
    order = rng.permutation(n_pages).astype(I32)
    table, at = np.full((len(lens), width), -1, I32), 0
    for i, n in enumerate(lens):
        held = min(-(-max(int(n), 0) // page), width)
        table[i, :held] = order[at:at + held]
        at += held
    free = np.full(n_pages, -1, I32)
    free[:n_pages - at] = order[at:]
    return table, free, n_pages - at


def _check_plan(lens, new, page, width, n_pages, tokens, count=None, seed=0, with_refs=True):
    rng = np.random.default_rng(seed)
    table, free, there = _tables(rng, lens, page, width, n_pages)
    count = there if count is None else count
    refs = np.zeros(n_pages, I32)
    want = ref.plan(lens, new, table, free, count, n_pages, page, tokens, refs if with_refs else None)
    d_table, d_refs = up(table), up(refs) if with_refs else None
    got = ta.PagedPlan(page).eval(ints(lens), ints(new), d_table, up(free), ints([count]), tokens, refs=d_refs)
    for name in ("lens", "starts", "slots", "positions", "free_count", "refused"):
        np.testing.assert_array_equal(got[name].to_numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(d_table.to_numpy(), want["table"])
    if with_refs:
        np.testing.assert_array_equal(d_refs.to_numpy(), want["refs"])
    return want


@pytest.mark.parametrize("n,longest,most,page", [(1, 0, 1, 16), (1, 100, 1, 1), (3, 40, 5, 7), (64, 500, 1, 16), (257, 300, 9, 32), (1500, 90, 3, 16), (4096, 40, 2, 5), (70, 2000, 300, 64)])
def test_plan(rt, n, longest, most, page):
    rng = np.random.default_rng(n)
    lens, new = rng.integers(0, longest, n, endpoint=True), rng.integers(0, most, n, endpoint=True)
    width = -(-(longest + most) // page) + 1
    n_pages = int(sum(-(-(a + b) // page) for a, b in zip(lens, new))) + 3
    for tokens in {int(new.sum()), int(new.sum()) + 11}:
        assert _check_plan(lens, new, page, width, n_pages, tokens, seed=n)["refused"][0] == 0
    _check_plan(lens, new, page, width, n_pages, int(new.sum()), seed=n, with_refs=False)


def test_plan_refuses_what_does_not_fit(rt):
    page, width = 4, 3
    lens, new = [3, 12, 4, 11, -1, 5, 5, 0, 8], [2, 1, 0, 1, 3, -2, 2, 9, 4]
    for count in (0, 1, 2, 4, 5, 6, 100, -3):
        for tokens in (0, 3, 8, 9, 18, 30):
            _check_plan(lens, new, page, width, 40, tokens, count=min(count, 20))
    assert _check_plan(lens, new, page, width, 40, 30)["refused"][0] == 3
    big = 1 << 30
    _check_plan([5, big, 2 ** 31 - 1, 7], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 1], page, width, 40, 30)      # (sums that would leave 32 bits)
    _check_plan([5, 2, 7], [big, 1, 1], page, width, 40, 30)


def test_plan_without_sequences_or_tokens(rt):
    _check_plan([], [], 16, 4, 8, 5)
    _check_plan([3, 4], [0, 0], 16, 4, 8, 0)
    _check_plan([0, 0], [0, 0], 16, 0, 0, 0)


def test_plan_over_holes_and_ids_that_are_no_pages(rt):
    """A partial page that is a hole gets no slots; free ids outside of the pool are handed out as they are, and stored for nobody."""
    page = 4
    table, free = np.array([[-1, -1, -1], [7, 99, -1]], I32), np.array([5, 400, -2, 6], I32)
    want = ref.plan([2, 6], [4, 4], table, free, 4, 10, page, 8, np.zeros(10, I32))
    free10 = np.full(10, -1, I32)
    free10[:4] = free
    d_table, refs = up(table), up(np.zeros(10, I32))
    got = ta.PagedPlan(page).eval(ints([2, 6]), ints([4, 4]), d_table, up(free10), ints([4]), 8, refs=refs)
    np.testing.assert_array_equal(got["slots"].to_numpy(), want["slots"])
    np.testing.assert_array_equal(d_table.to_numpy(), want["table"])
    np.testing.assert_array_equal(refs.to_numpy(), want["refs"])
    assert (want["slots"][:2] == -1).all() and want["slots"][2] == 6 * 4


# ---- append ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 64, 16), (5, 2, 128, 16), (33, 3, 7, 5), (700, 8, 128, 32), (64, 2, 63, 16), (9, 70, 2, 1), (3, 1, 2050, 4)])
def test_append(rt, dtype, tokens, heads, d, page):
    rng = np.random.default_rng(tokens)
    n_pages = tokens // page + 3
    pools = [rng.standard_normal((n_pages, heads, page, d)).astype(dtype) for _ in range(2)]
    rows = [rng.standard_normal((tokens, heads, d)).astype(dtype) for _ in range(2)]
    slots = rng.permutation(n_pages * page)[:tokens].astype(I32)
    slots[::7] = [-1, n_pages * page, 2 ** 31 - 1, -2 ** 31][tokens % 4]      # (nowhere)
    dk, dv = (up(p) for p in pools)
    ta.PagedAppend().eval(up(rows[0]), up(rows[1]), up(slots), dk, dv)
    for got, r, p in ((dk, rows[0], pools[0]), (dv, rows[1], pools[1])):
        assert got.to_numpy().tobytes() == ref.append(r, p, slots).tobytes()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,skew", [(128, 0), (64, 1), (66, 0), (64, 8)])
def test_append_of_views_into_pools_of_other_orders(rt, dtype, d, skew):
    """Rows of a fused projection, and pages laid out [n_pages, page, heads, head_dim] behind an offset."""
    rng, tokens, heads, page, n_pages = np.random.default_rng(5), 21, 3, 8, 6
    fused = rng.standard_normal((tokens, 9 * d + skew)).astype(dtype)
    size = fused.itemsize
    pools = [rng.standard_normal((n_pages, page, heads, d)).astype(dtype) for _ in range(2)]
    slots = rng.permutation(n_pages * page)[:tokens].astype(I32)
    base, dk, dv = up(fused), up(pools[0]), up(pools[1])
    view = lambda at: ta.DeviceTensor((tokens, heads, d), dtype, ptr=base.ptr.value + at * size, owner=base)  # noqa: E731
    shaped = lambda t: ta.DeviceTensor((n_pages, heads, page, d), dtype, ptr=t.ptr.value, owner=t)  # noqa: E731
    ta.PagedAppend().eval(view(3 * d), view(6 * d + skew), up(slots), shaped(dk), shaped(dv), k_strides=(9 * d + skew, d), v_strides=(9 * d + skew, d),
                          page_strides=(page * heads * d, d, heads * d))
    for got, at, p in ((dk, 3 * d, pools[0]), (dv, 6 * d + skew, pools[1])):
        rows = fused[:, at:at + 3 * d].reshape(tokens, heads, d)
        assert got.to_numpy().tobytes() == ref.append(rows, p.transpose(0, 2, 1, 3), slots).transpose(0, 2, 1, 3).tobytes()


# ---- attention -----------------------------------------------------------------------------------------------------


def _attend(rng, lens, hq, hkv, sq, d, page, dtype, width=None, garbage=True, holes=0.0, page_order="heads", scale=None, causal=True, spare=3, offset=0):
    lens = np.asarray(lens, I32)
    held = np.array([-(-max(int(n), 0) // page) for n in lens])
    width = int(held.max(initial=0)) if width is None else width
    n_pages = int(np.minimum(held, width).sum()) + spare
    order = rng.permutation(n_pages).astype(I32)
    table, at = rng.integers(-5, n_pages + 5, (len(lens), width)).astype(I32), 0      # (anything behind a sequence's pages)
    k, v = (rng.standard_normal((n_pages, hkv, page, d)).astype(dtype) for _ in range(2))
    used = np.zeros((n_pages, page), bool)
    for i, n in enumerate(lens):
        h = min(held[i], width)
        table[i, :h] = order[at:at + h]
        at += h
        for p in range(h):
            used[table[i, p], :max(0, int(n) - p * page)] = True
    if garbage:   # what belongs to no sequence may hold anything
        for pool in (k, v):
            pool.transpose(0, 2, 1, 3)[~used] = np.array([np.nan, np.inf, -np.inf])[rng.integers(0, 3, (int((~used).sum()), hkv, d))].astype(dtype)
    if holes:
        cut = rng.random(table.shape) < holes
        table[cut] = rng.choice([-1, n_pages, 2 ** 31 - 1, -2 ** 31], int(cut.sum()))
    q = (rng.standard_normal((len(lens), hq, sq, d)) * 2).astype(dtype)
    want, bound = ref.attend(q, k, v, table, lens, scale=scale, causal=causal)

    def pool(x):
        if page_order == "tokens":
            x = np.ascontiguousarray(x.transpose(0, 2, 1, 3))
        base = up(np.concatenate([np.zeros(offset, dtype), x.reshape(-1)]))
        return ta.DeviceTensor((n_pages, hkv, page, d), dtype, ptr=base.ptr.value + offset * x.itemsize, owner=base)

    strides = (hkv * page * d, d, hkv * d) if page_order == "tokens" else None
    out = up(np.full(q.shape, np.nan, dtype))
    got = ta.PagedSdpa(scale, is_causal=causal).eval(up(q), pool(k), pool(v), up(table.reshape(len(lens), width)), up(lens), out=out, page_strides=strides).to_numpy()
    assert_within(got, want, bound, f"{lens.tolist()[:6]} {hq}/{hkv} {sq} {d} {page} {np.dtype(dtype).name}")


HEADS = [(1, 1), (2, 1), (4, 1), (14, 2), (8, 8), (32, 2), (6, 2)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [16, 32, 48, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_lengths(rt, dtype, page, d):
    """Every length around a tile and a page, one after the other, and none."""
    rng = np.random.default_rng(page + d)
    _attend(rng, [1], 4, 2, 1, d, page, dtype)
    _attend(rng, [0], 4, 2, 1, d, page, dtype)
    _attend(rng, [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 0, 127, 128, 129, 130, 255, 256, 257], 4, 2, 1, d, page, dtype)
    _attend(rng, [2000, 0, 3, 777, 1, 1300], 8, 2, 1, d, page, dtype, width=2100 // page + 4)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attend_heads(rt, dtype, hq, hkv):
    rng = np.random.default_rng(hq)
    for d in (64, 128):
        _attend(rng, [300, 17, 0, 129], hq, hkv, 1, d, 16, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("sq", [2, 3, 5, 16, 17, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_several_queries(rt, dtype, sq, causal):
    """Sequences that hold fewer tokens than they have queries leave rows empty."""
    rng = np.random.default_rng(sq)
    _attend(rng, [sq, 300, sq - 1, 1, 0, 64, 65 + sq], 8, 2, sq, 128, 16, dtype, causal=causal, garbage=True)
    _attend(rng, [200, 1000], 14, 2, sq, 64, 32, dtype, causal=causal)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,page,offset", [(80, 16, 0), (128, 1, 0), (128, 7, 0), (64, 24, 0), (128, 16, 1), (64, 16, 4), (2, 3, 0), (2048, 4, 0), (1, 16, 0)])
def test_attend_any_size(rt, dtype, d, page, offset):
    rng = np.random.default_rng(d)
    _attend(rng, [0, 1, 40, 97], 4, 2, 1, d, page, dtype, offset=offset)
    _attend(rng, [5, 40], 4, 1, 3, d, page, dtype, offset=offset)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("sq", [1, 4])
@pytest.mark.parametrize("page", [16, 32, 64, 5])
def test_attend_over_holes(rt, dtype, sq, page):
    """Entries that are no pages hide their tokens; a sequence of holes alone is zeros."""
    rng = np.random.default_rng(page)
    _attend(rng, [500, 64, 33, 700, 1, 16], 8, 2, sq, 128, page, dtype, holes=0.4)
    _attend(rng, [500, 64, 1200], 8, 2, sq, 64, page, dtype, holes=0.95)
    _attend(rng, [500, 64], 8, 2, sq, 64, page, dtype, holes=1.0)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_pages_in_token_order(rt, dtype):
    rng = np.random.default_rng(3)
    for d, page in ((128, 16), (64, 64), (64, 9)):
        _attend(rng, [300, 0, 1, 95, 600], 8, 2, 1, d, page, dtype, page_order="tokens")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_many_sequences(rt, dtype):
    rng = np.random.default_rng(4)
    _attend(rng, rng.integers(0, 90, 400), 8, 2, 1, 64, 16, dtype)
    _attend(rng, rng.integers(0, 20, 3000), 2, 1, 1, 64, 16, dtype)
    _attend(rng, [0] * 300 + [3] + [0] * 300, 4, 2, 1, 64, 16, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_long(rt, dtype):
    rng = np.random.default_rng(6)
    _attend(rng, [20011], 4, 2, 1, 128, 16, dtype)
    _attend(rng, [9000, 1, 12000, 0, 8000], 4, 1, 2, 64, 64, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_lengths_that_the_table_has_no_pages_for(rt, dtype):
    """Taken as the nearest that it has."""
    rng = np.random.default_rng(7)
    _attend(rng, [100, -5, 2 ** 31 - 1, 64, -2 ** 31], 4, 2, 1, 64, 16, dtype, width=4)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_scales_and_sizes_of_scores(rt, dtype):
    rng = np.random.default_rng(8)
    _attend(rng, [300, 40], 4, 2, 1, 128, 16, dtype, scale=3.0)
    _attend(rng, [300, 40], 4, 2, 1, 64, 16, dtype, scale=0.0)
    _attend(rng, [300, 40], 4, 2, 1, 64, 16, dtype, scale=-1.0)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_rows_that_are_not_numbers_stay_so(rt, dtype, d):
    """A query of NaN is the row that shows it; a value of NaN that is seen shows in every row that sees it."""
    rng = np.random.default_rng(9)
    lens, page = [3000, 40], 16
    n_pages = 188 + 3
    table = np.full((2, 188), -1, I32)
    table[0], table[1, :3] = np.arange(188), [188, 189, 190]
    q, k, v = (rng.standard_normal(s).astype(dtype) for s in ((2, 4, 1, d), (n_pages, 2, page, d), (n_pages, 2, page, d)))
    clean = ta.PagedSdpa().eval(up(q), up(k), up(v), up(table), ints(lens)).to_numpy()
    q[0, 1, 0, 3] = np.nan
    v[189, 1, 5, 7] = np.nan
    got = ta.PagedSdpa().eval(up(q), up(k), up(v), up(table), ints(lens)).to_numpy()
    assert np.isnan(got[0, 1]).all() and np.isnan(got[1, 2:, 0, 7]).all()
    for at in (np.s_[0, 0], np.s_[0, 2:], np.s_[1, :2]):
        assert got[at].tobytes() == clean[at].tobytes()


# ---- sequences that go on from others -----------------------------------------------------------------------------------


def _check_reorder(parents, table, lens, refs, free, count, page):
    want = ref.reorder(parents, table, lens, refs, free, count, page)
    got = ta.PagedReorder(page).eval(ints(parents), up(table), up(lens), up(refs), up(free), ints([count]))
    for name, w in want.items():
        np.testing.assert_array_equal(got[name].to_numpy(), w, err_msg=name)
    return want


@pytest.mark.parametrize("n,longest,page,spare", [(1, 20, 16, 2), (4, 100, 16, 10), (9, 50, 4, 9), (64, 300, 16, 70), (257, 60, 7, 300), (3000, 30, 8, 3000), (12, 9000, 1, 40000)])
def test_reorder(rt, n, longest, page, spare):
    """Several steps one after the other, each from what the last one left; places without a parent among them."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, longest, n, endpoint=True).astype(I32)
    width, n_pages = -(-longest // page) + 1, int((-(-lens // page)).sum()) + spare
    table, free, count = _tables(rng, lens, page, width, n_pages)
    refs = np.zeros(n_pages, I32)
    refs[table[table >= 0]] = 1
    for step in range(4):
        parents = rng.integers(-1 if step % 2 else 0, n, n)
        if step == 2:
            parents = np.arange(n)
        w = _check_reorder(parents, table, lens, refs, free, count, page)
        assert w["missing"][0] == 0
        table, lens, refs, free, count = w["table"], w["lens"], w["refs"], w["free_pages"], int(w["free_count"][0])
        held = np.bincount(table[table >= 0], minlength=n_pages)
        np.testing.assert_array_equal(held, refs)          # every page is held, or free, exactly once
        assert sorted(free[:count]) == list(np.flatnonzero(held == 0))


def test_reorder_without_enough_free_pages_changes_nothing(rt):
    rng = np.random.default_rng(1)
    lens = np.array([5, 9, 3], I32)
    table, free, count = _tables(rng, lens, 4, 4, 8)
    refs = np.zeros(8, I32)
    refs[table[table >= 0]] = 1
    w = _check_reorder([0, 0, 0], table, lens, refs, free, 1, 4)
    assert w["missing"][0] == 1
    _check_reorder([0, 0, 0], table, lens, refs, free, 2, 4)
    _check_reorder([7, -1, -9], table, lens, refs, free, 2, 4)


def test_reorder_of_pages_that_others_hold_and_of_holes(rt):
    """A partial page that has another holder is copied for all children; holes and ids that are no pages stay where they are."""
    table = np.array([[0, 1, 2, -1], [0, 1, 3, -1], [5, -1, 4, -1], [6, 99, -1, -1]], I32)
    lens, refs = np.array([10, 11, 9, 7], I32), np.array([2, 2, 2, 1, 1, 1, 1, 0, 0, 0, 0, 0], I32)
    free = np.array([7, 8, 9, 10, 11] + [-1] * 7, I32)
    for parents in ([0, 0, 1, 2], [3, 3, 2, 0], [0, 1, 2, 3], [-1, -1, -1, -1], [2, 2, 2, 2]):
        _check_reorder(parents, table, lens, refs, free, 5, 4)


def test_reorder_of_nothing(rt):
    empty, none = np.zeros((0, 3), I32), np.zeros(0, I32)
    _check_reorder([], empty, none, np.ones(5, I32), np.full(5, -1, I32), 0, 4)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,d,page,pools", [(1, 64, 16, 1), (8, 128, 16, 4), (3, 7, 5, 2), (70, 2, 4, 2), (2, 64, 16, 300)])
def test_copy(rt, dtype, heads, d, page, pools):
    rng, n_pages = np.random.default_rng(page), 12
    host = [rng.standard_normal((n_pages, heads, page, d)).astype(dtype) for _ in range(pools)]
    copies = np.array([[0, 1, 3], [0, 2, page], [4, 3, 1], [-1, -1, 0], [5, n_pages, 2], [n_pages, 6, 2], [7, 8, 0], [9, 10, page + 5]], I32)
    device = [up(h) for h in host]
    ta.PagedCopy().eval(up(copies), device)
    for got, h in zip(device, host):
        assert got.to_numpy().tobytes() == ref.copy(h, copies).tobytes()
    ta.PagedCopy().eval(up(copies[:0]), device)
    ta.PagedCopy().eval(up(copies), [])


# ---- arguments that the Python side looks at ---------------------------------------------------------------------------------


def test_shapes_and_types_are_refused(rt):
    q, k, t, n = up(np.zeros((2, 4, 1, 64), F16)), up(np.zeros((5, 2, 16, 64), F16)), ints(np.zeros((2, 3))), ints([1, 1])
    op = ta.PagedSdpa()
    for bad in ((up(np.zeros((2, 4, 64), F16)), k, k, t, n), (q, k, up(np.zeros((5, 2, 16, 32), F16)), t, n), (up(np.zeros((2, 4, 1, 32), F16)), k, k, t, n), (up(np.zeros((2, 4, 1, 64), F32)), k, k, t, n),
                (q, k, k, ints(np.zeros((3, 3))), n), (q, k, k, t, ints([1])), (q, k, k, up(np.zeros((2, 3), F32)), n), (up(np.zeros((2, 3, 1, 64), F16)), k, k, t, n)):
        with pytest.raises(ta.TractRocmError):
            op.eval(*bad)
    with pytest.raises(ta.TractRocmError):
        op.eval(q, k, k, t, n, out=up(np.zeros((2, 4, 1, 64), F32)))
    with pytest.raises(ta.TractRocmError):
        ta.PagedPlan(16).eval(n, ints([1]), t, ints([0] * 5), ints([5]), 2)
    with pytest.raises(ta.TractRocmError):
        ta.PagedPlan(16).eval(n, n, t, ints([0] * 5), ints([5]), 2, out={"slots": ints([0, 0, 0])})
    with pytest.raises(ta.TractRocmError):
        ta.PagedAppend().eval(up(np.zeros((3, 2, 32), F16)), up(np.zeros((3, 2, 32), F16)), ints([0, 1, 2]), k, k)
    with pytest.raises(ta.TractRocmError):
        ta.PagedCopy().eval(ints([[0, 1, 2]]), [k, up(np.zeros((5, 2, 16, 64), F32))])
    with pytest.raises(ta.TractRocmError):
        ta.PagedReorder(16).eval(n, t, n, ints([0] * 5), ints([0] * 4), ints([5]))
    refs = ints([0] * 5)
    plan = ta.PagedPlan(16)
    plan.eval(n, n, t, ints([0] * 5), ints([5]), 2, refs=refs)
    with pytest.raises(ta.TractRocmError):   # (a type that changes from call to call)
        plan.eval(n, n, t, ints([0] * 5), ints([5]), 2, refs=up(np.zeros(5, np.int64)))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,sq,causal", [(70, 16, 8, 9, True), (40, 24, 8, 14, True), (70, 24, 8, 12, False), (70, 16, 8, 40, True)])
def test_attend_several_tiles_of_rows(rt, dtype, d, n, hq, hkv, sq, causal):
    """17 to 32, 33 to 64 and more rows of a kv head, in so many sequences that units of the most row tiles, or half as many, fill the workgroups."""
    rng = np.random.default_rng(n + sq)
    lens = rng.integers(0, 60, n)
    lens[:3] = 300, 0, 129
    _attend(rng, lens, hq, hkv, sq, d, 16, dtype, causal=causal, holes=0.05)


def _later_tokens(rng, lens, hq, hkv, sq, d, page, dtype):
    n, width = len(lens), -(-int(lens.max()) // page)
    held = -(-lens // page)
    n_pages = int(held.sum())
    order, table, at = rng.permutation(n_pages).astype(I32), np.full((n, width), -1, I32), 0
    for i in range(n):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
    k, v = (rng.standard_normal((n_pages, hkv, page, d)).astype(dtype) for _ in range(2))
    q = rng.standard_normal((n, hq, sq, d)).astype(dtype)
    bad_k, bad_v, zero_k, zero_v = k.copy(), v.copy(), k.copy(), v.copy()
    seen, token = np.array([np.nan, np.inf, -np.inf]), np.full(n, -1)
    for i in range(n):
        token[i] = int(rng.integers(max(0, lens[i] - sq + 1), lens[i]))
        place = (table[i, token[i] // page], slice(None), token[i] % page)
        bad_v[place][:, 1:4], zero_v[place][:, 1:4] = seen.astype(dtype), 0
        bad_k[place][:, d - 1], zero_k[place] = np.nan, 0
    sees = (lens[:, None] - sq + np.arange(sq)[None, :] >= token[:, None])[:, None, :, None]
    run = lambda kk, vv: ta.PagedSdpa().eval(up(q), up(kk), up(vv), up(table), up(lens)).to_numpy()  # noqa: E731
    want, bound = ref.attend(q, k, zero_v, table, lens)
    got = run(k, bad_v)
    hit = np.broadcast_to(sees, got.shape).copy()
    hit[..., 0], hit[..., 4:] = False, False
    np.testing.assert_array_equal(got[hit], np.broadcast_to(np.concatenate([[0], seen, np.zeros(d - 4)]), got.shape)[hit].astype(dtype))
    assert_within(np.where(hit, want, got), want, bound, "values")
    want, bound = ref.attend(q, zero_k, zero_v, table, lens)
    got = run(bad_k, bad_v)
    hit = np.broadcast_to(sees, got.shape)
    assert np.isnan(got[hit]).all()
    assert_within(np.where(hit, want, got), want, bound, "keys")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("hq,hkv,sq,page", [(8, 8, 2, 16), (4, 1, 3, 32), (16, 2, 3, 16), (8, 2, 9, 16), (14, 2, 6, 64), (6, 3, 70, 16)])
def test_attend_later_tokens_that_are_not_numbers(rt, dtype, d, hq, hkv, sq, page):
    """An infinity or a NaN among the values of a call's own tokens is seen by the queries from its token on alone, and in its feature; a
    NaN among the keys makes those rows NaN.  Lengths of one step, of several parts, of fewer tokens than queries."""
    rng = np.random.default_rng(d + sq)
    lens = np.array([sq, 3, 150, 700, 127 + sq // 2, 2600, 20, 128], I32)
    _later_tokens(rng, lens, hq, hkv, sq, d, page, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,hkv,sq", [(64, 16, 8, 20), (64, 16, 8, 9), (128, 16, 8, 9)])
def test_attend_later_tokens_that_are_not_numbers_in_many_sequences(rt, dtype, d, hq, hkv, sq):
    """The same in units of several row tiles."""
    rng = np.random.default_rng(d * sq)
    lens = rng.integers(1, 50, 300).astype(I32)
    lens[:3] = 400, 129, 1
    _later_tokens(rng, lens, hq, hkv, sq, d, 16, dtype)


# ---- the far ends of what the calls allow -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_tables_of_so_many_tokens_that_a_launch_takes_one_sequence(rt, dtype, d):
    """Rows of the table for 2^30 tokens, 32 kv heads: a line of tiles counted in 31 bits has room for one sequence, whatever its length.
    Pages of 2^20 tokens of which 100 are used: heads lie 128 rows apart, inside of one another's pages."""
    rng, page, width, heads, lens = np.random.default_rng(d), 1 << 20, 1 << 10, 32, [100, 0, 33]
    apart = 128
    strides = (heads * apart * d, apart * d, d)
    size = 2 * strides[0] + (heads - 1) * strides[1] + page * d
    n_pages = 3
    used = [rng.standard_normal((n_pages, heads, apart, d)).astype(dtype) for _ in range(2)]
    pools = []
    for u in used:
        flat = np.zeros(size, dtype)
        flat[:u.size] = u.reshape(-1)
        base = up(flat)
        pools.append((base, ta.DeviceTensor((n_pages, heads, page, d), dtype, ptr=base.ptr.value, owner=base)))
    table = np.full((3, width), -1, I32)
    table[:, 0] = [2, 0, 1]
    q = (rng.standard_normal((3, heads, 1, d)) * 2).astype(dtype)
    got = ta.PagedSdpa().eval(up(q), pools[0][1], pools[1][1], up(table), ints(lens), page_strides=strides).to_numpy()
    want, bound = ref.attend(q, *used, table[:, :1], np.array(lens, I32))
    assert_within(got, want, bound, f"{d} {np.dtype(dtype).name}")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attend_more_rows_than_a_launch_has_workgroups(rt, dtype):
    """5120000 query rows of an odd size, a workgroup each: sequences of one token repeat its value, empty ones are zeros."""
    rng, n, heads, sq, d, page = np.random.default_rng(9), 5000, 8, 128, 2, 3
    k, v = (rng.standard_normal((n, 2, page, d)).astype(dtype) for _ in range(2))
    lens = rng.integers(0, 2, n).astype(I32)
    got = ta.PagedSdpa(is_causal=False).eval(up(np.zeros((n, heads, sq, d), dtype)), up(k), up(v), up(np.arange(n, dtype=I32)[:, None]), up(lens)).to_numpy()
    want = np.where(lens[:, None, None, None] > 0, np.repeat(v[:, :, 0], heads // 2, axis=1)[:, :, None, :], dtype(0))
    np.testing.assert_array_equal(got, np.broadcast_to(want, got.shape))


def test_append_more_tokens_than_a_launch_has_workgroups(rt):
    """4194304 workgroups of a token each, and 7 tokens more; most go nowhere.  Rows begin 8 elements apart."""
    tokens, heads, d, n_pages, page = (1 << 22) + 7, 8, 1024, 3, 4
    rng = np.random.default_rng(3)
    flat = rng.integers(0, 1 << 15, (tokens - 1) * 8 + heads * d, dtype=np.uint16).view(F16)
    slots = np.full(tokens, -1, I32)
    goes = [0, 5, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, tokens - 1]
    slots[goes] = [3, 11, 0, 7, 4, 8]
    base, pools = up(flat), [up(np.zeros((n_pages, heads, page, d), F16)) for _ in range(2)]
    rows = ta.DeviceTensor((tokens, heads, d), F16, ptr=base.ptr.value, owner=base)
    ta.PagedAppend().eval(rows, rows, up(slots), *pools, k_strides=(8, d), v_strides=(8, d))
    want = np.zeros((n_pages, heads, page, d), F16)
    for t in goes:
        want[slots[t] // page, :, slots[t] % page] = flat[t * 8:t * 8 + heads * d].reshape(heads, d)
    for pool in pools:
        assert pool.to_numpy().tobytes() == want.tobytes()


@pytest.mark.parametrize("causal", [True, False])
def test_attend_the_same_pages_many_times(rt, causal):
    """Sequences that are one another's copies, and a page that comes twice in a row of the table."""
    rng, d, page = np.random.default_rng(4), 128, 16
    k, v = (rng.standard_normal((4, 2, page, d)).astype(F16) for _ in range(2))
    table = np.array([[0, 1, 0, 2], [0, 1, 0, 2], [3, 3, 3, 3], [0, 1, 0, 2], [2, 2, 1, 1]], I32)
    lens = np.array([64, 64, 50, 1, 33], I32)
    q = (rng.standard_normal((5, 8, 3, d)) * 2).astype(F16)
    got = ta.PagedSdpa(is_causal=causal).eval(up(q), up(k), up(v), up(table), up(lens)).to_numpy()
    want, bound = ref.attend(q, k, v, table, lens, causal=causal)
    assert_within(got, want, bound, "shared")
    if not causal:
        one = ta.PagedSdpa(is_causal=False).eval(up(np.repeat(q[:1], 5, axis=0)), up(k), up(v), up(table), up(lens)).to_numpy()
        assert_within(one[1], one[0].astype(np.float64), 2 * bound[0], "copies")


@pytest.mark.parametrize("n_pages,page", [(20000, 1), (100000, 2), (1 << 20, 1)])
def test_reorder_of_large_pools(rt, n_pages, page):
    """More pages than a workgroup takes: the stack of the free ones is put together from several shares."""
    rng, n, longest = np.random.default_rng(n_pages), 40, min(n_pages // 50 * page, 8000)
    lens = rng.integers(0, longest, n).astype(I32)
    width = -(-longest // page)
    table, free, count = _tables(rng, lens, page, width, n_pages)
    refs = np.zeros(n_pages, I32)
    np.add.at(refs, table[table >= 0], 1)
    _check_reorder(rng.integers(-2, n + 2, n).astype(I32), table, lens, refs, free, count, page)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_pages_behind_eight_gibibytes(rt, dtype, order):
    """Byte and element offsets that pass 32 bits: the append, the copy and the attention over pages at both ends of a pool and around its middle."""
    rng, heads, d, page = np.random.default_rng(12), 8, 128, 16
    n_pages = (1 << 33) // (heads * d * page * np.dtype(dtype).itemsize) + 7
    pools = [ta.DeviceTensor((n_pages, heads, page, d), dtype) for _ in range(2)]
    strides = (heads * page * d, d, heads * d) if order == "tokens" else None
    ids = np.array([n_pages - 1, 0, n_pages // 2, n_pages // 2 - 1, n_pages - 3, n_pages // 4], I32)
    lens = np.array([40, 33], I32)
    table = ids.reshape(2, 3)
    rows = [rng.standard_normal((73, heads, d)).astype(dtype) for _ in range(2)]
    slots = np.concatenate([table[i, np.arange(n) // page] * page + np.arange(n) % page for i, n in enumerate(lens)]).astype(I32)
    ta.PagedAppend().eval(up(rows[0]), up(rows[1]), up(slots), *pools, page_strides=strides)

    q = (rng.standard_normal((2, 32, 1, d)) * 2).astype(dtype)
    small = [np.zeros((6, heads, page, d), dtype) for _ in range(2)]
    for x in range(2):
        for t, slot in enumerate(slots):
            small[x][int(np.flatnonzero(ids == slot // page)[0]), :, slot % page] = rows[x][t]
    want, bound = ref.attend(q, *small, np.arange(6, dtype=I32).reshape(2, 3), lens)
    got = ta.PagedSdpa().eval(up(q), *pools, up(table), up(lens), page_strides=strides).to_numpy()
    assert_within(got, want, bound, f"{order} {np.dtype(dtype).name}")

    copies = np.array([[n_pages - 1, n_pages - 2, page], [0, n_pages // 2 + 1, 9]], I32)
    ta.PagedCopy().eval(up(copies), pools, page_strides=strides)
    got = ta.PagedSdpa().eval(up(q), *pools, ints([[n_pages - 2, 0, n_pages // 2], [n_pages // 2 - 1, n_pages - 3, n_pages // 4]]), up(lens), page_strides=strides).to_numpy()
    assert_within(got, want, bound, f"copied, {order} {np.dtype(dtype).name}")
    one = ints([9, 9])
    got = ta.PagedSdpa().eval(up(q), *pools, ints([[n_pages // 2 + 1], [0]]), one, page_strides=strides).to_numpy()
    assert got[0].tobytes() == ta.PagedSdpa().eval(up(q[[0, 0]]), *pools, ints([[0], [0]]), one, page_strides=strides).to_numpy()[0].tobytes()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,sq,causal", [(300, 16, 8, 20, True), (300, 8, 8, 30, False), (160, 16, 8, 9, True)])
def test_attend_tiles_of_rows_in_many_sequences(rt, dtype, d, n, hq, hkv, sq, causal):
    """So many steps that no unit takes fewer row tiles than it can, or half as many."""
    rng = np.random.default_rng(n + sq)
    lens = rng.integers(0, 40, n)
    lens[:4] = 300, 0, 129, sq
    _attend(rng, lens, hq, hkv, sq, d, 16, dtype, causal=causal, holes=0.05)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_with_workspaces_of_every_size(rt, dtype, d):
    """That of the call, of fewer queries, a byte less than any, and none: all within the bounds, and nothing behind the workspace is written."""
    rng, n, hq, hkv, sq, page = np.random.default_rng(d), 300, 16, 8, 20, 16
    lens = rng.integers(0, 40, n).astype(I32)
    lens[:2] = 500, 129
    held = -(-lens // page)
    table, at = np.full((n, held.max()), -1, I32), 0
    for i in range(n):
        table[i, :held[i]] = np.arange(at, at + held[i])
        at += held[i]
    k, v = (rng.standard_normal((at, hkv, page, d)).astype(dtype) for _ in range(2))
    q = rng.standard_normal((n, hq, sq, d)).astype(dtype)
    want, bound = ref.attend(q, k, v, table, lens)
    sizes = []
    for queries in (20, 16, 9, 1):
        b = C.c_size_t()
        ta._lib.call("trocm_sdpa_paged_workspace_bytes", n, hq, hkv, queries, d, C.byref(b))
        sizes.append(b.value)
    assert sizes[0] >= sizes[1] >= sizes[2] >= sizes[3]
    dq, dk, dv, dt, dl = up(q), up(k), up(v), up(table), up(lens)
    for size in [*sizes, sizes[-1] - 1, 0]:
        ws, out = up(np.full(size + 4096, 0xA5, np.uint8)), up(np.full(q.shape, np.nan, dtype))
        if size:
            ta._lib.call("trocm_sdpa_workspace_init", ws.ptr, size, None)
        ta._lib.call("trocm_sdpa_paged", dq.ptr, 1 if dtype is F16 else 0, n, hq, hkv, sq, d, dk.ptr, dv.ptr, at, page, None, dt.ptr, table.shape[1], dl.ptr, out.ptr,
                     float("nan"), 1, ws.ptr if size else None, size, None)
        assert_within(out.to_numpy(), want, bound, f"{size} bytes")
        assert (ws.to_numpy()[size:] == 0xA5).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,sq,page,causal", [(400, 8, 8, 1, 16, True), (400, 6, 3, 1, 32, True), (300, 8, 8, 3, 16, False), (500, 9, 3, 5, 16, True), (200, 32, 16, 1, 48, True)])
def test_attend_many_short_sequences(rt, dtype, d, n, hq, hkv, sq, page, causal):
    """More units of a step than workgroups: a wave each where sequences have up to 64 keys, beside longer ones and empty ones."""
    rng = np.random.default_rng(n + hq + sq)
    lens = rng.integers(0, 70, n)
    lens[rng.random(n) < 0.1] = 0
    lens[:4] = 64, 65, 32, 200
    _attend(rng, lens, hq, hkv, sq, d, page, dtype, causal=causal, holes=0.1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_later_tokens_that_are_not_numbers_in_short_sequences(rt, dtype, d):
    rng = np.random.default_rng(d)
    _later_tokens(rng, rng.integers(1, 64, 400, endpoint=True).astype(I32), 8, 4, 5, d, 16, dtype)
