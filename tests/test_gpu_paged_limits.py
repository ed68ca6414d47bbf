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
