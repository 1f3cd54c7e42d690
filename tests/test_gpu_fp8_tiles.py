"""8-bit products of many rows, in each form of tile that they take: what lies behind the matrices reaches nothing, captured calls and calls that share the
library's scratch give what they give alone. Tolerances are those of test_gpu_fp8.py."""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, ops, pack_f32, unpack_f32
from tests import fp8_reference as ref
from tests.hip_graph import Graph
from tests.test_gpu_fp8 import _tolerance, _weights
from tests.test_gpu_gated_delta import Case

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]
# 128 x 64 tiles (twice), 128 x 128 ones, 256 x 256 ones that are all cut in two, some of them, none (with lower halves behind the last row), and f32's. K ends
# inside a block and inside a window of four blocks' scales, and N inside a tile.
SHAPES = [(129, 5600, 400), (300, 4200, 656), (100, 33000, 144), (400, 8300, 144), (4100, 4360, 144), (2600, 4700, 272)]


def _tiled(dt, m, n, k):
    rc, launches, _, _ = ops.plan("fp8_qmm", dt, 8, 128, m, n, k)
    return rc == 0 and launches[0][3] > 64 * 1024   # (stages of both operands: the kernels of few rows have a few KB)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_nan_stays_in_its_row_and_column(dt, m, n, k):
    print(f"[case] fp8_qmm {dt.name} M{m} N{n} K{k} with NaN", flush=True)
    assert _tiled(dt, m, n, k)
    rng = np.random.default_rng(m)
    w, ws = _weights(rng, n, k)
    x, xs = ref.quantize(rng.standard_normal((m, k)).astype(np.float32), 1)
    clean = ref.values(x, xs, 1), ref.values(w, ws, 128)
    w[7, k - 1] = w[n - 1, 0] = 127
    x[m - 1, 3], x[130 % m, k - 1] = 255, 127
    xs[5, -1] = np.nan
    ws[2, 0] = np.nan
    rows, cols = [m - 1, 130 % m, 5], [7, n - 1, *range(256, 384)]
    want = clean[0] @ clean[1].T
    fine = np.ones((m, n), bool)
    fine[rows] = False
    fine[:, cols] = False
    behind = 300 * k
    wb, xb = (GpuBuffer.from_bytes(v.tobytes() + b"\x7f" * behind) for v in (w, x))
    wsb, xsb = (GpuBuffer.from_bytes(v.tobytes() + b"\xff" * 65536) for v in (ws, xs))
    size = m * n * dt.size_bytes
    out = GpuBuffer.from_bytes(b"\xa5" * (size + 4096))
    ops.fp8_qmm(dt, wb, wsb, xb, xsb, out, m, n, k)
    raw = out.read_bytes()
    got = unpack_f32(raw[:size], dt).reshape(m, n)
    assert raw[size:] == b"\xa5" * 4096
    assert np.array_equal(np.isnan(got), ~fine)
    assert np.all(np.abs(got - want)[fine] <= _tolerance(*clean, want, dt, k)[fine])


class _Product:
    def __init__(self, dt, m, n, k, seed):
        rng = np.random.default_rng(seed)
        self.dt, self.shape, self.m, self.k = dt, (m, n, k), m, k
        w, ws = _weights(rng, n, k)
        self.w, self.ws, self.x, self.out = GpuBuffer.from_bytes(w.tobytes()), GpuBuffer.from_bytes(ws.tobytes()), GpuBuffer(m * k * dt.size_bytes), GpuBuffer(m * n * dt.size_bytes)
        self.put(seed)

    def put(self, seed):
        self.x.upload(pack_f32(np.random.default_rng(seed).standard_normal(self.m * self.k).astype(np.float32), self.dt))

    def call(self):
        ops.fp8_qmv(self.dt, self.w, self.ws, self.x, self.out, *self.shape)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_captured(dt, m, n, k):
    assert _tiled(dt, m, n, k)
    p = _Product(dt, m, n, k, 1)
    g = Graph()
    try:
        with g:
            p.call()
        for turn in range(3):
            p.put(turn)
            p.out.upload(b"\xff" * p.out.nbytes)
            g.replay()
            first = p.out.read_bytes()
            p.call()
            assert p.out.read_bytes() == first and np.isfinite(unpack_f32(first, dt)).all()
    finally:
        g.close()


def test_calls_one_behind_the_other_share_scratch():
    """Products of each form of tile and a prompt through the delta rule, whose codes and chunks lie in the same buffer, without a wait between them."""
    products = [_Product(DTYPES[i % 3], *shape, i) for i, shape in enumerate(SHAPES)]
    delta = Case(DType.BF16, [700, 40], 2, 4, 128, 64)
    calls, outs = [p.call for p in products] + [delta.call], [p.out for p in products] + [delta.y, delta.state_out]
    for c in calls:
        c()
        ops.sync()
    want = [b.read_bytes() for b in outs]
    for order in ([0, 6, 1, 2, 6, 3, 5, 4], [5, 4, 3, 2, 6, 1, 0], [2, 0, 4, 1, 6, 3, 5]):
        for b in outs:
            b.zero()
        for i in order * 2:
            calls[i]()
        assert [b.read_bytes() for b in outs] == want, order
