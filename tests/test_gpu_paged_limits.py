"""The ends of what the entry points over pages take: sums of additions at 2^30 packed rows; K and V pages in one another's gaps."""
import numpy as np
import pytest

import tract_amd as ta
from tests import paged_ref as ref
from tests.attention_ref import assert_within
from tests.gpu_util import rt  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32
up = ta.DeviceTensor.from_numpy


def test_packed_rows_that_do_not_suffice_at_the_end_of_their_range(rt):
    """2^30 packed rows, of which a sequence that is refused for its pages leaves the next one 5: that one asks for 10, which its page has room for, and is
    refused; one that asks for nothing behind it is not."""
    top, page = 1 << 30, 16
    lens, new = [0, 3, 7, 2], [top - 5, 10, 0, 1]
    table, free = np.array([[-1, -1], [4, -1], [5, -1], [6, -1]], I32), np.full(9, -1, I32)
    d_table = up(table)
    got = ta.PagedPlan(page).eval(up(np.array(lens, I32)), up(np.array(new, I32)), d_table, up(free), up(np.zeros(1, I32)), top)
    assert got["refused"].to_numpy()[0] == 3 and got["free_count"].to_numpy()[0] == 0
    assert got["lens"].to_numpy().tolist() == lens and got["starts"].to_numpy().tolist() == [0, top - 5, top, top, top]
    np.testing.assert_array_equal(d_table.to_numpy(), table)
    for name in ("slots", "positions"):
        for at in (0, top // 2, top - 64):
            assert (ta.DeviceTensor((64,), I32, ptr=got[name].ptr.value + 4 * at, owner=got[name]).to_numpy() == -1).all(), (name, at)


LAYOUTS = {   # (order of pages, halves, heads and tokens in memory)
    "halves of a page": ("p2ht", lambda h, n, d: (2 * h * n * d, n * d, d), lambda h, n, d: h * n * d),
    "halves of a token": ("pt2h", lambda h, n, d: (2 * h * n * d, d, 2 * h * d), lambda h, n, d: h * d),
    "halves of a head": ("ph2t", lambda h, n, d: (2 * h * n * d, 2 * n * d, d), lambda h, n, d: n * d),
    "halves of a row": ("pht2", lambda h, n, d: (2 * h * n * d, 2 * n * d, 2 * d), lambda h, n, d: d),
}


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("first", ["k", "v"])
def test_pages_of_keys_and_values_in_one_tensor(rt, dtype, layout, first):
    """Appended, copied and attended over; what no slot names stays."""
    rng, n_pages, heads, page, d = np.random.default_rng(4), 7, 5, 16, 64
    order, strides, half = LAYOUTS[layout]
    strides, half = strides(heads, page, d), half(heads, page, d)
    pool = rng.standard_normal((2, n_pages, heads, page, d)).astype(dtype)     # 2, p, h, t
    axes = [{"2": 0, "p": 1, "h": 2, "t": 3}[x] for x in order] + [4]
    base = up(np.ascontiguousarray(pool.transpose(axes)))
    at = lambda i: ta.DeviceTensor((n_pages, heads, page, d), dtype, ptr=base.ptr.value + i * half * pool.itemsize, owner=base)  # noqa: E731
    k_at, v_at = (0, 1) if first == "k" else (1, 0)
    rows = [rng.standard_normal((20, heads, d)).astype(dtype) for _ in range(2)]
    slots = rng.permutation(n_pages * page)[:20].astype(I32)
    ta.PagedAppend().eval(up(rows[0]), up(rows[1]), up(slots), at(k_at), at(v_at), page_strides=strides)
    pool[k_at], pool[v_at] = ref.append(rows[0], pool[k_at], slots), ref.append(rows[1], pool[v_at], slots)
    copies = np.array([[2, 5, 9], [1, 6, 16], [-1, -1, 0]], I32)
    ta.PagedCopy().eval(up(copies), [at(0), at(1)], page_strides=strides)
    pool[0], pool[1] = ref.copy(pool[0], copies), ref.copy(pool[1], copies)
    assert base.to_numpy().tobytes() == np.ascontiguousarray(pool.transpose(axes)).tobytes()
    q, table, lens = rng.standard_normal((2, 10, 1, d)).astype(dtype), np.array([[0, 5, 3], [6, 2, -1]], I32), np.array([41, 20], I32)
    want, bound = ref.attend(q, pool[k_at], pool[v_at], table, lens)
    assert_within(ta.PagedSdpa().eval(up(q), at(k_at), at(v_at), up(table), up(lens), page_strides=strides).to_numpy(), want, bound, layout)


def test_pools_that_do_meet_are_refused(rt):
    """Half of a page apart where a page's tokens are not those of a half, a row apart, and halves that are longer than their gaps."""
    n_pages, heads, page, d = 4, 2, 16, 64
    base = up(np.zeros(4 * n_pages * heads * page * d, F16))
    at = lambda i: ta.DeviceTensor((n_pages, heads, page, d), F16, ptr=base.ptr.value + i * 2, owner=base)  # noqa: E731
    rows, slots, whole = up(np.zeros((3, heads, d), F16)), up(np.zeros(3, I32)), heads * page * d
    for by, strides in ((whole // 2, (2 * whole, page * d, d)), (d, (2 * whole, page * d, d)), (whole, None), (whole, (2 * whole - d, page * d, d)), (2 * whole, (2 * whole, page * d, d)),
                        (d, (2 * whole, 2 * d, 2 * heads * d - d)), (0, (2 * whole, page * d, d))):
        for a, b in ((0, by), (by, 0)):
            with pytest.raises(ta.TractRocmError, match="overlaps"):
                ta.PagedAppend().eval(rows, rows, slots, at(a), at(b), page_strides=strides)
