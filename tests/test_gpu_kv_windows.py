"""Windows that hide nothing: as long as a sequence may be and longer, up to what 32 bits hold (-1 from a caller that means none). The same bits as without one, whatever
the library's buffers held before."""
import numpy as np
import pytest

from metaltile_amd import DType
from tests.kv_reference import DTYPES
from tests.test_gpu_kv_attention import Attention, option  # noqa: F401

pytestmark = pytest.mark.gpu
PAST_31_BITS = [(1 << 31) - 1, 1 << 31, (1 << 31) + 77, (1 << 32) - 300, (1 << 32) - 1, -1]


def _called(c, window, before):
    before.call()
    c.out.upload(b"\xa5" * c.out.nbytes)
    c.window = window
    c.call()
    return c.out.read_bytes()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("kernel", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("lens,rows", [([500, 1, 90], [130, 1, 20]), ([500, 333, 90], [1, 2, 1])], ids=str)
def test_windows_that_hide_nothing(dt, kernel, lens, rows, option):  # noqa: F811
    """New rows behind a prefix in the cache; other keys and values in the scratch from the call before."""
    print(f"[case] kv_attention windows {dt.name} {lens} {rows} kernel {kernel}", flush=True)
    c = Attention(dt, lens, rows, width=40)
    before = Attention(dt, [512, 512, 512], [100, 100, 100], width=40, seed=7)
    option("kv.kernel", kernel)
    for slices in (0, 3):
        option("kv.slices", slices)
        want = _called(c, 0, before)
        c.hold(kernel)
        for window in [40 * 16] + PAST_31_BITS:
            assert _called(c, window, before) == want, window
        for window in (max(lens), 40 * 16 - 1):   # (they see as much; a shorter bound may cut them otherwise)
            _called(c, window, before)
            c.hold(kernel)


@pytest.mark.parametrize("kernel", [0, 1, 3])
@pytest.mark.parametrize("seqs", [40, 200, 512])
def test_many_sequences(kernel, seqs, option):  # noqa: F811
    rng = np.random.default_rng(seqs)
    lens = [int(n) for n in rng.integers(0, 300, seqs)]
    rows = [int(n) for n in rng.integers(0, 3, seqs)]
    c = Attention(DType.BF16, lens, rows, hq=2, hkv=1)
    before = Attention(DType.BF16, lens, rows, hq=2, hkv=1, seed=8)
    option("kv.kernel", kernel)
    for slices in (0, 4):
        option("kv.slices", slices)
        want = _called(c, 0, before)
        c.hold(kernel)
        for window in [c.pool.max_len] + PAST_31_BITS:
            assert _called(c, window, before) == want, window
