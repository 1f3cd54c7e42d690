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
