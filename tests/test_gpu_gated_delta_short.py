"""Batches of sequences around the length from which they go in chunks, many of them shorter: where each sequence's chunks lie in the scratch goes by
tokens or by sequences, whichever takes less. Against 64 bits, with the tolerances of test_gpu_gated_delta.py."""
import numpy as np
import pytest

from metaltile_amd import DType, _lib
from metaltile_amd.runtime import _ensure_init
from tests.test_gpu_gated_delta import Case

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]
_mixed = np.random.default_rng(3)
LENS = {"two_each": [2] * 100, "seventeen": [17] * 90, "one_chunk_among_many": [1] * 150 + [40] + [1] * 150, "around": [16, 17, 18, 0, 63, 64, 65, 1] * 12,
        "any": [int(n) for n in _mixed.integers(0, 70, 130)], "few_long": [int(n) for n in np.where(_mixed.random(150) < 0.08, _mixed.integers(60, 260, 150), _mixed.integers(0, 5, 150))],
        "long_last": [3] * 80 + [300], "long_first": [300] + [3] * 80}


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("most_kb", [0, 400])
@pytest.mark.parametrize("lens", LENS)
def test_short_sequences(dt, lens, most_kb):
    print(f"[case] gated_delta_rule {dt.name} {lens} most_kb{most_kb}", flush=True)
    lib = _ensure_init()
    c = Case(dt, LENS[lens], 1, 2, 64, 32, tail=5)
    _lib.check(lib.mtq_set_option(b"scratch.most_kb", most_kb))
    try:
        c.call()
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
    c.hold()


@pytest.mark.parametrize("each", [17, 32, 33, 48, 64, 65])
def test_equal_lengths(each):
    c = Case(DType.BF16, [each] * 70, 1, 2, 64, 32, equal=True)
    c.call()
    c.hold()
