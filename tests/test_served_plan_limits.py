"""Sizes next to what a launch can have, and past it: fewer than 2^32 threads along each dimension of a grid. A call is refused before any of its launches,
or goes another way; decided by shapes, so without a device."""
import numpy as np
import pytest

from metaltile_amd import DType, ops

OK, SHAPE = 0, -3
DTYPES = [DType.F32, DType.F16, DType.BF16]


def _fits(rc, launches):
    assert rc in (OK, SHAPE) and (rc == OK) == bool(launches)
    for name, grid, block, lds in launches:
        assert all(0 < g * b < 1 << 32 for g, b in zip(grid, block)), (name, grid, block)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_gated_delta_rule(dt):
    plan = lambda seqs, tokens, hk=16, hv=32, dk=128, dv=128: ops.plan("gated_delta_rule", dt, 0, dv, hk, hv, dk, seqs, tokens)
    rng = np.random.default_rng(4)
    for _ in range(300):
        seqs, hk = int(2 ** rng.uniform(8, 32)), int(rng.choice([1, 2, 16]))
        rc, launches, _, _ = plan(seqs, min(0xFFFFFFFF, int(seqs * 2 ** rng.uniform(0, 8))), hk, hk * int(rng.integers(1, 4)), dv=int(rng.choice([1, 128, 65536])))
        _fits(rc, launches)
    # More columns than the walk can have workgroups: token by token. More heads than that has: refused, and so are numbers of sequences that 32 bits
    # could not be counted up to in steps of 64.
    rc, launches, scratch, _ = plan(30000, 60000)
    assert rc == OK and [l[2] for l in launches] == [(256, 1, 1)] and scratch == 0
    rc, launches, scratch, _ = plan(20000, 40000)
    assert rc == OK and launches[1][2][0] >= 512 and scratch > 0
    assert plan((1 << 19) - 1, 1 << 19)[0] == OK and plan(1 << 19, 1 << 19)[0] == SHAPE
    for seqs in (1 << 24, (1 << 30) + 1, (1 << 31) - 1, 0xFFFFFFFF):
        assert plan(seqs, 0xFFFFFFFF, hk=1, hv=1, dk=1, dv=1)[0] == SHAPE


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("op", ["fp8_qmm", "fp8_qmv"])
def test_fp8_products(dt, op):
    plan = lambda m, n, k: ops.plan(op, dt, 8, 128, m, n, k)
    rng = np.random.default_rng(5)
    for _ in range(2000):
        m, n = (int(2 ** rng.uniform(0, hi)) for hi in ((8, 30), (30, 8), (30, 30))[int(rng.integers(3))])
        _fits(*plan(m, n, 16 * int(2 ** rng.uniform(0, 26)))[:2])
    most = (1 << 28) - 16
    for m, n in ((1, most), (2, most), (33, most), (128, most), (129, most), (512, most), (1 << 20, 1 << 17), (1 << 28, 16), (1 << 28, 128), (1 << 28, 129), (1 << 28, 512)):
        rc, launches, _, _ = plan(m, n, 16)
        _fits(rc, launches)
        assert rc == (SHAPE if op == "fp8_qmv" and m == 1 << 28 else OK)   # (as many blocks of x are more than the quantiser can have)
    for m, n, k in ((1, most + 1, 16), ((1 << 30) + 1, 16, 16), (1 << 22, 16, (1 << 22) + 16), (1 << 27, 1 << 27, 16)):
        rc, launches, _, _ = plan(m, n, k)
        assert rc == SHAPE and not launches
    if op == "fp8_qmm":   # more rows of w where tiles take them
        assert plan(100, 1 << 29, 16)[0] == (OK if dt == DType.F32 else SHAPE) and plan(200, 1 << 30, 16)[0] == (SHAPE if dt == DType.F32 else OK)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_fp8_quantize(dt):
    plan = lambda rows, cols, block: ops.plan("fp8_quantize", dt, 8, block, rows, 0, cols)
    rng = np.random.default_rng(6)
    for _ in range(500):
        _fits(*plan(int(2 ** rng.uniform(0, 30)), 16 * int(2 ** rng.uniform(0, 26)), int(rng.choice([1, 128])))[:2])
    assert plan((1 << 28) - 16, 128, 1)[0] == OK and plan(1 << 28, 128, 1)[0] == SHAPE
    assert plan(1 << 30, 128, 128)[0] == OK and plan(1 << 30, 256, 128)[0] == SHAPE


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_token_logprobs(dt):
    plan = lambda rows, vocab: ops.plan("token_logprobs", dt, 0, 0, rows, vocab, 1)
    rng = np.random.default_rng(7)
    for _ in range(500):
        _fits(*plan(int(2 ** rng.uniform(0, 32)), int(2 ** rng.uniform(0, 30)))[:2])
    assert plan((1 << 24) - 1, 100)[0] == OK and plan(1 << 24, 100)[0] == SHAPE


@pytest.mark.parametrize("dt,slot", [(DType.BF16, 2.0), (DType.F16, 2.8), (DType.F32, 3.6)], ids=lambda v: getattr(v, "name", None))
def test_short_sequences_reserve_scratch_by_their_tokens(dt, slot):
    """A chunk's slot has (16 heads x 3 operands x 64 x 128 terms of 16 bits, 32 heads x 37 KB) about 2 MB in bf16. Only a sequence of 17 tokens or more
    takes any, so a call has at most one for each 17 of its tokens, however many sequences it has, and makes its two launches once."""
    for seqs, tokens in ((256, 512), (64, 128), (1000, 1040), (4096, 8192)):
        rc, launches, scratch, count = ops.plan("gated_delta_rule", dt, 0, 128, 16, 32, 128, seqs, tokens)
        slots = tokens // 17 + 1
        assert rc == OK and scratch <= min(slots * slot * (1 << 20), 1 << 30)
        assert count == 2 * -(-slots // int((1 << 30) / (slot * (1 << 20))))
    # Prompts: a slot for each 64 tokens, and one for each sequence.
    _, _, scratch, _ = ops.plan("gated_delta_rule", dt, 0, 128, 16, 32, 128, 2, 4096)
    assert scratch <= (4096 // 64 + 2) * slot * (1 << 20)
