"""Residual addition, RMS norm and 8-bit output against 64 bits.

The sum is to the bit (one f32 addition, one rounding). y: a sum of squares in f32, at most cols / 8 + 16 roundings one after the other in a lane and over lanes (half of it in the root), and six
more roundings: rel = (cols / 16 + 16) 2^-24 at most. A scale is max |y| / 448, so rel + 2^-24 off; a code is the nearest e4m3 value to a quotient that is 2 rel + 2^-24 off: half a step
(2^-4 of the quotient from 2^-6 on, 2^-10 below) and that.
"""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, ops, pack_f32, unpack_f32
from tests import fp8_reference as fp8
from tests.hip_graph import Graph
from tests.kv_reference import DTYPES, typed

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Norm:
    def __init__(self, dt, rows, cols, residual=True, seed=1):
        self.dt, self.rows, self.cols = dt, rows, cols
        rng = self.rng = np.random.default_rng(seed + rows + cols)
        self.x = typed(rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1))), dt)
        self.r = typed(4 * rng.standard_normal((rows, cols)), dt) if residual else None
        self.w = typed(1 + 0.3 * rng.standard_normal(cols), dt)
        self.upload()

    def upload(self):
        up = GpuBuffer.from_bytes
        self.xb, self.wb = up(pack_f32(self.x, self.dt)), up(pack_f32(self.w, self.dt))
        self.rb = None if self.r is None else up(pack_f32(self.r, self.dt))
        n, b = self.rows * self.cols, fp8.blocks(self.cols)
        self.sum, self.codes, self.scales = up(b"\xa5" * (n * self.dt.size_bytes + 64)), up(b"\xa5" * (n + 64)), up(b"\xa5" * (4 * self.rows * b + 64))

    def call(self, sum_out="sum"):
        ops.add_rms_norm_fp8(self.dt, self.xb, self.rb, self.wb, EPS, self.sum if sum_out == "sum" else sum_out, self.codes, self.scales, self.rows, self.cols)

    def outputs(self):
        n, b = self.rows * self.cols, fp8.blocks(self.cols)
        for buf, size in ((self.codes, n), (self.scales, 4 * self.rows * b)):
            assert buf.read_bytes()[size:] == b"\xa5" * 64
        return np.frombuffer(self.codes.read_bytes(n), np.uint8).reshape(self.rows, self.cols), np.frombuffer(self.scales.read_bytes(4 * self.rows * b), "<f4").reshape(self.rows, b)

    def h(self):
        return self.x if self.r is None else (self.x + self.r).astype(np.float32)

    def hold(self, sum_buf="sum"):
        codes, scales = self.outputs()
        h = self.h()
        if sum_buf is not None:
            buf = self.sum if sum_buf == "sum" else sum_buf
            assert buf.read_bytes(h.size * self.dt.size_bytes) == pack_f32(h, self.dt)
        h = h.astype(np.float64) if self.r is None else self.x.astype(np.float64) + self.r.astype(np.float64)
        y = h * self.w.astype(np.float64) / np.sqrt((h * h).mean(1, keepdims=True) + EPS)
        rel = (self.cols / 16 + 16) * 2.0 ** -24
        cols = np.arange(self.cols) // 128
        most = np.stack([np.abs(y[:, cols == b]).max(1) for b in range(scales.shape[1])], 1)
        want = np.where(most > 0, np.maximum(most / 448, 2.0 ** -126), 1.0)
        assert np.all(np.abs(scales - want) <= (rel + 2.0 ** -23) * want)
        q = y / want[:, cols]
        got = fp8.e4m3_values()[codes].astype(np.float64)
        half = np.maximum(np.abs(q) * 2.0 ** -4, 2.0 ** -10)
        assert np.all(np.abs(got - q) <= half * (1 + 2.0 ** -10) + (2 * rel + 2.0 ** -22) * np.abs(q))


SHAPES = [(1, 16), (1, 128), (3, 144), (5, 1024), (4, 1040), (1, 4096), (33, 4144), (2, 8192), (7, 8208), (1, 16384), (2, 40000), (1, 65536), (2, 65552), (1, 100000), (300, 512), (129, 2048)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm(dt, rows, cols):
    print(f"[case] add_rms_norm_fp8 {dt.name} {rows}x{cols}", flush=True)
    c = Norm(dt, rows, cols)
    c.call()
    c.hold()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,cols", [(3, 144), (2, 4096), (2, 70000)])
def test_other_ways(dt, rows, cols):
    """Without a residual; the sum in the residual's place, in x's, or not at all: the same codes."""
    c = Norm(dt, rows, cols, residual=False)
    c.call()
    c.hold()
    c = Norm(dt, rows, cols)
    c.call()
    want = [x.tobytes() for x in c.outputs()]
    for where in (None, "residual", "x"):
        c.upload()
        buf = {"residual": c.rb, "x": c.xb, None: None}[where]
        c.call(buf)
        c.hold(buf)
        assert [x.tobytes() for x in c.outputs()] == want
        if where is None:
            assert c.sum.read_bytes() == b"\xa5" * c.sum.nbytes


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("cols", [256, 4096, 70000])
def test_rows_of_their_own(dt, cols):
    """Zeros: zeros (of the weight's sign) under a scale of 1. A NaN or an infinity stays in its row."""
    c = Norm(dt, 6, cols)
    c.x[1], c.r[1] = 0, 0
    c.x[2, 7] = np.nan
    c.r[3, cols - 1] = np.inf
    c.x[4, :] = 0
    c.r[4, :] = 0
    c.x[4, 3] = 5.0
    c.upload()
    c.call()
    codes, scales = c.outputs()
    assert np.all((codes[1] & 127) == 0) and np.all(scales[1] == 1)
    value = fp8.e4m3_values()[codes].astype(np.float64) * scales[:, np.arange(cols) // 128]
    assert np.all(np.isnan(value[2])) and np.isnan(value[3, cols - 1])
    keep = [0, 1, 4, 5]
    c.x, c.r, c.rows = c.x[keep], c.r[keep], 4
    c.sum, c.codes, c.scales = (GpuBuffer.from_bytes(v) for v in (pack_f32(c.h(), dt), codes[keep].tobytes() + b"\xa5" * 64, scales[keep].tobytes() + b"\xa5" * 64))
    c.hold()


def test_the_next_product_takes_it():
    """Codes and scales are fp8_qmm's activations: against the quantiser's own of the same y in f32."""
    c = Norm(DType.F32, 20, 512, residual=False)
    c.w[:] = 1
    c.upload()
    c.call()
    codes, scales = c.outputs()
    y = (c.x * (1 / np.sqrt((c.x.astype(np.float64) ** 2).mean(1, keepdims=True) + EPS))).astype(np.float32)
    wc, ws = fp8.quantize(y, 1)
    assert np.allclose(ws, scales, rtol=1e-6) and (codes == wc).mean() > 0.999


def test_captured():
    c = Norm(DType.BF16, 5, 4096)
    g = Graph()
    try:
        with g:
            c.call()
        assert g.nodes == 1
        for turn in range(3):
            c.x = typed(c.rng.standard_normal(c.x.shape), c.dt)
            c.xb.upload(pack_f32(c.x, c.dt))
            g.replay()
            c.hold()
    finally:
        g.close()


def test_refusals():
    c = Norm(DType.BF16, 2, 128)

    def refused(code, dt=c.dt, x=c.xb, r=c.rb, w=c.wb, eps=EPS, s=c.sum, codes=c.codes, scales=c.scales, rows=2, cols=128):
        with pytest.raises(MtqError) as e:
            ops.add_rms_norm_fp8(dt, x, r, w, eps, s, codes, scales, rows, cols)
        assert e.value.code == code

    refused(-2, dt=3)
    for what in ("x", "w", "codes", "scales"):
        refused(-2, **{what: 0})
    refused(-2, x=c.xb.ptr + 2)
    refused(-2, r=c.rb.ptr + 8)
    refused(-2, s=c.sum.ptr + 4)
    refused(-2, codes=c.codes.ptr + 8)
    refused(-2, scales=c.scales.ptr + 2)
    refused(-3, cols=24)
    refused(-3, cols=0)
    refused(-3, rows=1 << 28)
    refused(-2, eps=-1.0)
    refused(-2, eps=float("nan"))
    ops.add_rms_norm_fp8(c.dt, 0, None, 0, EPS, None, 0, 0, 0, 128)
    assert c.codes.read_bytes() == b"\xa5" * c.codes.nbytes
