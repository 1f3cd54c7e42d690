"""Attention over the paged 4-bit cache: the length of each row's error, and of a whole call's, against what its roundings add up to (kv_precision)."""
import numpy as np
import pytest

from metaltile_amd import DType
from tests import kv_precision
from tests.kv_reference import DTYPES
from tests.test_gpu_kv_attention import Attention, option  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = [  # lens, rows, options
    ([300], [200], dict(window=17)), ([300, 70], [200, 70], dict(window=64, dim=64)), ([300], [200], dict(window=64, dim=256, group=32, hq=2, hkv=1)),
    ([200], [77], dict(group=128, hq=2, hkv=2)), ([200, 33, 1], [200, 20, 1], dict(dim=64, group=32, hq=4, hkv=1)), ([700], [130], dict(hq=6, hkv=2)), ([900, 400], [70, 70], dict(dim=256, group=128, hq=4, hkv=1)),
    ([2500], [100], dict(hq=2, hkv=1)), ([900, 40, 333], [1, 1, 4], dict(hq=32, hkv=8)), ([400], [1], dict(dim=256, group=64, hq=8, hkv=1))]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("kernel,slices", [(0, 0), (1, 1), (1, 3), (2, 1), (2, 4), (3, 3), (4, 1), (4, 3)], ids=str)
def test_lengths_of_errors(dt, kernel, slices, option):  # noqa: F811
    option("kv.kernel", kernel)
    option("kv.slices", slices)
    for lens, rows, more in CASES:
        print(f"[case] kv_attention precision {dt.name} kernel {kernel} slices {slices} {lens} {rows} {more}", flush=True)
        c = Attention(dt, lens, rows, seed=5, **more)
        c.call()
        want, each, of_all = kv_precision.attention(c.pool, c.q, c.offsets, c.hq, c.scale, c.window, dt, c.rounded(kernel))
        off = c.result() - want
        far = np.linalg.norm(off, axis=2)
        assert np.all(far <= each), f"{(far / each).max()} of a row's bound"
        if want.shape[0] * want.shape[1] >= 100:
            assert np.linalg.norm(off) <= of_all, f"{np.linalg.norm(off) / of_all} of the whole bound, {np.linalg.norm(off) / np.linalg.norm(want)} of the result"
