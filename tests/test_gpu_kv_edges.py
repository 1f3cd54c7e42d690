"""Calls that the paged cache's documentation allows: a capacity far above all lengths, queries that a call without query heads does not look at."""
import numpy as np
import pytest

from metaltile_amd import ops
from tests.kv_reference import DTYPES
from tests.test_gpu_kv_attention import Attention, option  # noqa: F401
from tests.test_gpu_kv_cache import Append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("kernel", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("lens,rows", [([1000, 0, 40, 333], [1, 1, 2, 1]), ([700, 0, 90], [100, 3, 90])], ids=str)
def test_a_capacity_far_above_all_lengths(dt, kernel, lens, rows, option):  # noqa: F811
    print(f"[case] kv_attention capacity {dt.name} {lens} {rows} kernel {kernel}", flush=True)
    option("kv.kernel", kernel)
    for window in (0, 100):
        c = Attention(dt, lens, rows, width=8192, window=window)
        assert c.pool.max_len == 131072
        for slices in (0, 5):
            option("kv.slices", slices)
            c.out.upload(b"\xa5" * c.out.nbytes)
            c.call()
            c.hold(kernel)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_queries_that_no_head_has(dt):
    """hq 0: queries and their strides are not looked at, whatever they are."""
    c = Append(dt, [12, 2, 30], [5, 2, 7])
    before = c.q_out.read_bytes()
    for q, q_out, stride in ((c.at[0], c.at[0], None), (c.at[0] + 2, c.q_out.ptr + 2, 3), (None, c.q_out, 0), (c.q_out, c.q_out, 5)):
        ops.kv_append(dt, c.pool.cache, c.batch, c.at[1], c.at[2], row_stride=c.strides, q=q, q_out=q_out, hq=0, q_out_stride=stride, cos_sin=c.tb, n_positions=c.table.shape[0], rot=c.rot)
    c.want()
    for got, want in zip(c.pool.downloaded(), c.pool.parts):
        assert all(np.array_equal(g, w, equal_nan=True) for g, w in zip(got, want))
    assert c.q_out.read_bytes() == before
