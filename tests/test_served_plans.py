"""What the 8-bit floating point calls, the gated delta rule and the log probabilities would launch, and what they refuse: decided
by shapes, so without a device."""
import numpy as np
import pytest

from metaltile_amd import DType, ops

OK, BAD_ARG, SHAPE = 0, -2, -3
DTYPES = [DType.F32, DType.F16, DType.BF16]


def _check(launches):
    assert launches
    for name, grid, block, lds in launches:
        assert name and 0 < block[0] * block[1] * block[2] <= 1024 and block[0] % 64 == 0
        assert 0 < grid[0] <= 0x7FFFFFFF and 0 < grid[1] <= 65535 and grid[2] == 1 and lds <= 160 * 1024


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_fp8(dt):
    rng = np.random.default_rng(1)
    for _ in range(300):
        m, n, k = int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 17)), 16 * int(2 ** rng.uniform(0, 11))
        for op in ("fp8_qmm", "fp8_qmv"):
            rc, launches, scratch, count = ops.plan(op, dt, 8, 128, m, n, k)
            assert rc == OK and count == len(launches)
            _check(launches)
        for block in (1, 128):
            rc, launches, scratch, _ = ops.plan("fp8_quantize", dt, 8, block, m, 0, k)
            assert rc == OK and scratch == 0 and len(launches) == 1
            _check(launches)


@pytest.mark.parametrize("op", ["fp8_qmm", "fp8_qmv"])
def test_fp8_refusals(op):
    assert ops.plan(op, DType.BF16, 8, 128, 4, 64, 100)[0] == SHAPE
    assert ops.plan(op, DType.BF16, 8, 128, 4, 64, 0)[0] == SHAPE
    assert ops.plan(op, DType.BF16, 8, 128, 4, 0, 128)[0] == SHAPE
    assert ops.plan(op, DType.BF16, 8, 128, 4, 64, 0xFFFFFFF0)[0] == SHAPE
    assert ops.plan(op, DType.BF16, 8, 128, 4, 0xFFFFFFFF, 128)[0] == SHAPE
    assert ops.plan(op, DType.BF16, 8, 128, 0xFFFFFFFF, 64, 128)[0] == SHAPE
    assert ops.plan(op, 3, 8, 128, 4, 64, 128)[0] == BAD_ARG
    assert ops.plan(op, DType.BF16, 8, 128, 0, 64, 128) == (OK, [], 0, 0)


def test_fp8_quantize_refusals():
    assert ops.plan("fp8_quantize", DType.BF16, 8, 64, 4, 0, 128)[0] == BAD_ARG
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 4, 0, 24)[0] == SHAPE
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 4, 0, 0)[0] == SHAPE
    assert ops.plan("fp8_quantize", 7, 8, 1, 4, 0, 128)[0] == BAD_ARG
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 0, 0, 128) == (OK, [], 0, 0)
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 1 << 30, 0, 1 << 30)[0] == SHAPE   # 2^53 blocks
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 0xFFFFFFFF, 0, 128)[0] == SHAPE
    assert ops.plan("fp8_quantize", DType.BF16, 8, 1, 1, 0, 0xFFFFFFF0)[0] == SHAPE


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_gated_delta_rule(dt):
    rng = np.random.default_rng(2)
    for _ in range(300):
        hk = int(rng.integers(1, 17))
        hv, dk, dv = hk * int(rng.integers(1, 4)), int(rng.choice([1, 20, 64, 100, 128, 256])), int(rng.choice([1, 24, 64, 128, 200, 512]))
        seqs = int(2 ** rng.uniform(0, 9))
        tokens = seqs * int(2 ** rng.uniform(0, 12))
        rc, launches, _, count = ops.plan("gated_delta_rule", dt, 0, dv, hk, hv, dk, seqs, tokens)
        assert rc == OK and min(count, 8) == len(launches)   # (two launches for each window of chunks)
        _check(launches)


def test_gated_delta_rule_refusals():
    plan = lambda hk=2, hv=4, dk=128, dv=128, seqs=1, tokens=4, dt=DType.BF16: ops.plan("gated_delta_rule", dt, 0, dv, hk, hv, dk, seqs, tokens)[0]
    assert plan() == OK
    assert plan(hk=3) == SHAPE and plan(hk=0) == SHAPE and plan(hv=0) == SHAPE
    assert plan(dk=0) == SHAPE and plan(dk=257) == SHAPE and plan(dv=0) == SHAPE and plan(dv=65537) == SHAPE
    assert plan(dt=5) == BAD_ARG
    assert plan(seqs=1 << 31, hk=1, hv=1) == SHAPE
    assert ops.plan("gated_delta_rule", DType.BF16, 0, 128, 2, 4, 128, 0, 0) == (OK, [], 0, 0)
    assert plan(tokens=0) == OK   # states are passed on


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_token_logprobs(dt):
    rng = np.random.default_rng(3)
    for _ in range(300):
        rows, vocab, top = int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 18)), int(rng.integers(0, 33))
        top = min(top, vocab)
        rc, launches, scratch, count = ops.plan("token_logprobs", dt, 0, 0, rows, vocab, top)
        assert rc == OK and count == len(launches) and (scratch > 0) == (count == 2)
        _check(launches)


def test_token_logprobs_refusals():
    assert ops.plan("token_logprobs", DType.BF16, 0, 0, 1, 100, 33)[0] == SHAPE
    assert ops.plan("token_logprobs", DType.BF16, 0, 0, 1, 8, 9)[0] == SHAPE
    assert ops.plan("token_logprobs", DType.BF16, 0, 0, 1, 0, 0)[0] == SHAPE
    assert ops.plan("token_logprobs", DType.BF16, 0, 0, 1, (1 << 30) + 1, 0)[0] == SHAPE
    assert ops.plan("token_logprobs", 9, 0, 0, 1, 100, 1)[0] == BAD_ARG
    assert ops.plan("token_logprobs", DType.BF16, 0, 0, 0, 100, 1) == (OK, [], 0, 0)
