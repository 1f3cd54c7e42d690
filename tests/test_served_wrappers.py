"""What ops.gated_delta_rule hands to the library for each way to give its arguments; without a device."""
import numpy as np
import pytest

from metaltile_amd import DType, ops


class _Library:
    def mtq_gated_delta_rule(self, *args):
        self.args = args
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(ops, "_ensure_init", lambda: lib)
    return lib


@pytest.mark.parametrize("stride,want", [(None, (256, 256, 512)), (1024, (1024,) * 3), (np.int64(1024), (1024,) * 3), (np.uint32(1024), (1024,) * 3), ((300, 301, 600), (300, 301, 600)),
                                         ([300, 301, 600], (300, 301, 600)), (np.array([300, 301, 600]), (300, 301, 600))], ids=str)
def test_row_stride(library, stride, want):
    ops.gated_delta_rule(DType.BF16, 1, 2, 3, 4, 5, None, 7, 8, 1, 4, 2, 4, 128, 128, row_stride=stride)
    assert library.args[1:7] == (1, want[0], 2, want[1], 3, want[2])


def test_without_tokens(library):
    ops.gated_delta_rule(DType.BF16, None, None, None, None, None, 6, 7, None, 2, 0, 2, 4, 128, 128)
    assert library.args[1:14] == (None, 256, None, 256, None, 512, None, None, None, None, 6, 7, None)
