"""Which calls of the attention over the 4-bit cache are cut into slices, by the launches that they would take: decided by sizes, so without a device."""
import pytest

from metaltile_amd import DType, ops


def _cut(dt, seqs, longest, new=1, dim=128, hq=32, hkv=8):
    rc, launches, scratch, _ = ops.plan("kv_attention", dt, longest, 64, hq, hkv, dim, seqs, seqs * new)
    assert rc == 0 and launches
    assert (len(launches) == 2) == (scratch > 0)   # (the second joins the slices' sums)
    return len(launches) == 2


@pytest.mark.parametrize("dt,new,dim", [(DType.F32, 1, 128), (DType.F16, 4, 128), (DType.BF16, 4, 128), (DType.BF16, 4, 64), (DType.F32, 1, 64)], ids=str)
def test_sequences_that_may_be_long_are_cut(dt, new, dim):
    """One that is long ends alone where none is cut, also when there are three workgroups to each compute unit."""
    for longest in (4096, 6000, 8192, 20000):
        assert _cut(dt, 96, longest, new, dim) and _cut(dt, 128, longest, new, dim)
    assert not _cut(dt, 128, 1000, new, dim) and not _cut(dt, 500, 2048, new, dim)
    assert not _cut(dt, 256, 8192, new, dim)


@pytest.mark.parametrize("dt", [DType.F16, DType.BF16], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_four_rows(dt, dim):
    cut = lambda seqs, longest: _cut(dt, seqs, longest, dim=dim)  # noqa: E731
    assert cut(128, 6000) and cut(96, 8192)
    assert not cut(128, 4096) and not cut(300, 1000) and not cut(256, 8192)
