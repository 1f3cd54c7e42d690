"""8-bit products of a few activation rows where the library's buffer cannot be had: rows are quantised in LDS, with the same results."""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32
from metaltile_amd.runtime import _ensure_init
from tests.test_gpu_fp8 import _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [DType.F32, DType.F16, DType.BF16], ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", [(1, 40, 40960), (2, 5000, 512), (4, 4112, 400), (5, 300, 2000), (9, 33, 128), (16, 257, 1040), (16, 100, 9856), (3, 16, 400)])
def test_few_rows(dt, m, n, k):
    print(f"[case] fp8_qmv {dt.name} M{m} N{n} K{k} without scratch", flush=True)
    rng = np.random.default_rng(m + n + k)
    w, ws = _weights(rng, n, k)
    wb, wsb, xb = GpuBuffer.from_bytes(w.tobytes()), GpuBuffer.from_bytes(ws.tobytes()), GpuBuffer.from_bytes(pack_f32(rng.standard_normal((m, k)).astype(np.float32), dt))
    size = m * n * dt.size_bytes
    out = GpuBuffer(size + 64)
    lib, got = _ensure_init(), []
    for most_kb in (0, 1):
        out.upload(b"\xff" * (size + 64))
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", most_kb))
        try:
            assert (ops.plan("fp8_qmv", dt, 8, 128, m, n, k)[2] == 0) or not most_kb
            ops.fp8_qmv(dt, wb, wsb, xb, out, m, n, k)
        finally:
            _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
        got.append(out.read_bytes())
    assert got[0] == got[1] and got[0][size:] == b"\xff" * 64


def test_more_rows_than_fit():
    b = GpuBuffer(1 << 20)
    lib = _ensure_init()
    _lib.check(lib.mtq_set_option(b"scratch.most_kb", 1))
    try:
        for m, k in ((17, 128), (16, 9872)):
            with pytest.raises(MtqError):
                ops.fp8_qmv(DType.BF16, b, b, b, b, m, 16, k)
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
