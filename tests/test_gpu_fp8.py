"""8-bit floating point in blocks of 128: the quantiser to the bit, products against 64 bits.

Tolerance of a product: codes' products are exact in f32 (4 + 4 bits); a block's sum has 128 terms, at most 128 roundings of 2^-24 of the sum of
their magnitudes; its scale is a product rounded once and the block's share a multiply-add: 2 x 2^-24; K / 128 blocks in f32, again 2^-24 each of the
sum of magnitudes at most; at the end one rounding to the type, half a step of the value (an f16 below 2^-14: 2^-25). For f16 and bf16 results the matrix
cores line up eight neighbouring products by the largest and drop what lies below 2^-13 of its power of two: up to 2^-13 of the largest for each of
the seven others, and the largest is at most the product of the eight codes' largest on either side. That is the bound of one value; over all values the
2-norm of the error has to stay below 0.6 half steps (a rounding's is 1 / sqrt(3)) plus 4e-5 of the result's.
"""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests import fp8_reference as ref
from tests.hip_graph import Graph

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]
HALF_STEP = {DType.F32: 2.0 ** -24, DType.F16: 2.0 ** -11, DType.BF16: 2.0 ** -8}


def _typed(x, dt):
    return unpack_f32(pack_f32(x, dt), dt).reshape(x.shape)


def _same_codes(got, want):
    nan = (want & 127) == 127
    return np.array_equal(got[~nan], want[~nan]) and np.all((got[nan] & 127) == 127)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (3, 144), (7, 2048), (127, 256), (128, 128), (130, 400), (300, 1008), (1, 16384)])
def test_quantize(dt, block, rows, cols):
    print(f"[case] fp8_quantize {dt.name} block{block} {rows}x{cols}", flush=True)
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1)))).astype(np.float32)
    x[:, cols // 2] *= 30
    x = _typed(x, dt)
    codes, scales = ref.quantize(x, block)
    xb, cb, sb = GpuBuffer.from_bytes(pack_f32(x, dt)), GpuBuffer.from_bytes(b"\xa5" * (codes.size + 64)), GpuBuffer.from_bytes(b"\xa5" * (4 * scales.size + 64))
    ops.fp8_quantize(dt, xb, cb, sb, rows, cols, block)
    assert np.array_equal(np.frombuffer(sb.read_bytes(4 * scales.size), "<f4").reshape(scales.shape), scales)
    assert np.array_equal(np.frombuffer(cb.read_bytes(codes.size), np.uint8).reshape(codes.shape), codes)
    assert cb.read_bytes()[codes.size:] == b"\xa5" * 64 and sb.read_bytes()[4 * scales.size:] == b"\xa5" * 64


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_values_of_their_own(block):
    """Every e4m3 value and the ties between them (scale 1), zeros, the smallest numbers, infinities and NaN."""
    finite = np.sort(ref.e4m3_values()[np.isfinite(ref.e4m3_values())])
    ties = (finite[1:] + finite[:-1]) / 2
    all_of = np.concatenate([finite, ties, np.nextafter(ties.astype(np.float32), np.float32(1e9)), np.nextafter(ties.astype(np.float32), np.float32(-1e9))]).astype(np.float32)
    x = np.zeros((136, 128), np.float32)
    n = -(-all_of.size // 127)
    for i in range(n):
        part = all_of[i * 127:(i + 1) * 127]
        x[i, :part.size] = part
        x[i, 127] = 448
    if block == 1:
        x[n:n + 1] = 1e-45
        x[n + 1, 5], x[n + 1, 6] = 1e-38, -1e-45
        x[n + 2, 3], x[n + 2, 4], x[n + 2, 5] = np.inf, 1.0, -np.inf
        x[n + 3, 3], x[n + 3, 4], x[n + 3, 5] = np.nan, 1.0, -3.0
        x[n + 4] = 3.4028235e38
        x[n + 5] = np.nan
    codes, scales = ref.quantize(x, block)
    xb, cb, sb = GpuBuffer.from_bytes(x.tobytes()), GpuBuffer(x.size), GpuBuffer(4 * scales.size)
    ops.fp8_quantize(DType.F32, xb, cb, sb, *x.shape, block)
    assert np.array_equal(np.frombuffer(sb.read_bytes(), "<f4").reshape(scales.shape), scales)
    assert _same_codes(np.frombuffer(cb.read_bytes(), np.uint8).reshape(codes.shape), codes)


@pytest.mark.parametrize("lo,hi", [(-20, 20), (-149, -60), (60, 118)])
def test_quotients_beside_ties(lo, hi):
    """Elements whose quotients lie on the middle between two codes, or up to two f32 steps beside it, under scales of any mantissa: the f32
    quotient is the correctly rounded one, and so is the code. Blocks of the smallest scales, which are divided by in another way, too."""
    rng = np.random.default_rng(hi + 200)
    finite = np.sort(ref.e4m3_values()[np.isfinite(ref.e4m3_values())])
    ties = (finite[1:] + finite[:-1]) / 2
    x = np.zeros((4096, 128), np.float32)
    most = (448 * (1 + rng.random(4096)) * 2.0 ** rng.integers(lo, hi, 4096)).astype(np.float32)
    with np.errstate(all="ignore"):
        scale = np.maximum(most / np.float32(448), np.float32(2.0 ** -126)).astype(np.float64)
        v = (rng.choice(ties, x.shape) * scale[:, None]).astype(np.float32)
        for _ in range(2):
            v = np.where(rng.random(x.shape) < 0.4, np.nextafter(v, np.where(rng.random(x.shape) < 0.5, np.float32(np.inf), np.float32(-np.inf))), v)
    x[:] = np.clip(v, -most[:, None], most[:, None])
    x[:, 7] = most
    x[:, 9], x[:, 11] = -0.0, 0.0
    codes, scales = ref.quantize(x, 1)
    xb, cb, sb = GpuBuffer.from_bytes(x.tobytes()), GpuBuffer(x.size), GpuBuffer(4 * scales.size)
    ops.fp8_quantize(DType.F32, xb, cb, sb, *x.shape, 1)
    assert np.array_equal(np.frombuffer(sb.read_bytes(), "<f4").reshape(scales.shape), scales)
    assert np.array_equal(np.frombuffer(cb.read_bytes(), np.uint8).reshape(codes.shape), codes)


def _weights(rng, n, k):
    codes = ref.e4m3_codes(np.clip(64 * rng.standard_normal((n, k)), -448, 448))
    return codes, (1e-3 * (0.5 + rng.random((ref.blocks(n), ref.blocks(k))))).astype(np.float32)


def _tolerance(x, w, want, dt, k):
    terms = np.abs(x) @ np.abs(w).T
    tol = (128 + k // 128 + 4) * 2.0 ** -24 * terms + HALF_STEP[dt] * np.abs(want) + (2.0 ** -25 if dt == DType.F16 else 0)
    if dt != DType.F32:
        xg, wg = (np.abs(v).reshape(v.shape[0], -1, 8).max(2) for v in (x, w))
        tol += 7 * 2.0 ** -13 * (xg @ wg.T)
    return tol


SHAPES = [(1, 1, 16), (1, 16, 128), (1, 130, 144), (2, 64, 256), (3, 17, 512), (5, 257, 1040), (8, 100, 4096), (16, 128, 384), (16, 33, 2000), (17, 300, 640), (31, 129, 128),
          (33, 512, 1024), (48, 200, 272), (64, 64, 512), (65, 384, 896), (77, 1000, 1536), (128, 256, 256), (129, 511, 400), (200, 900, 2048), (256, 256, 128), (257, 700, 1168),
          (300, 1300, 640), (513, 260, 304)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(dt, m, n, k):
    print(f"[case] fp8 product {dt.name} M{m} N{n} K{k}", flush=True)
    rng = np.random.default_rng(m + n + k)
    w, ws = _weights(rng, n, k)
    x = _typed((rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float32), dt)
    codes, scales = ref.quantize(x, 1)
    xv, wv = ref.values(codes, scales, 1), ref.values(w, ws, 128)
    want = xv @ wv.T
    tol = _tolerance(xv, wv, want, dt, k)
    wb, wsb, xb, cb, sb = (GpuBuffer.from_bytes(v) for v in (w.tobytes(), ws.tobytes(), pack_f32(x, dt), codes.tobytes(), scales.tobytes()))
    size = m * n * dt.size_bytes
    out = GpuBuffer.from_bytes(b"\xff" * (size + 64))
    results = []
    for call in (lambda: ops.fp8_qmm(dt, wb, wsb, cb, sb, out, m, n, k), lambda: ops.fp8_qmv(dt, wb, wsb, xb, out, m, n, k)):
        out.upload(b"\xff" * (size + 64))
        call()
        raw = out.read_bytes()
        assert raw[size:] == b"\xff" * 64
        got = unpack_f32(raw[:size], dt).reshape(m, n).astype(np.float64)
        assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) / tol))
        assert m * n < 1000 or np.linalg.norm(got - want) <= (0.6 * HALF_STEP[dt] + (4e-5 if dt != DType.F32 else 1e-6)) * np.linalg.norm(want)
        results.append(raw)
    assert m > 16 or np.allclose(unpack_f32(results[0][:size], dt), unpack_f32(results[1][:size], dt), rtol=2 * HALF_STEP[dt], atol=float(tol.max()))


# More tiles than the CUs take as groups of rows: 128 x 128, 128 x 64, 256 x 256, those cut in two (with a lower half behind the last row), f32 as well.
TILED = [(40, 16500, 272), (129, 4112, 400), (300, 4200, 656), (65, 8200, 1168), (400, 8300, 144), (2600, 4700, 272), (4100, 4360, 400), (130, 8300, 784)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", TILED)
def test_products_in_tiles(dt, m, n, k):
    test_products(dt, m, n, k)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("m,n,k", [(129, 4112, 400), (300, 4200, 656), (400, 8300, 144), (2600, 4700, 272), (4100, 4360, 144), (130, 8300, 400)])
def test_exact_in_tiles(dt, m, n, k):
    """Codes of -1, 0 and 1 and scales of 1: every sum is a whole number, which bf16 holds up to 256."""
    rng = np.random.default_rng(m)
    wi, xi = rng.integers(-1, 2, (n, k)), rng.integers(-1, 2, (m, k)) * (rng.random((m, k)) < 0.1)
    w, x = ref.e4m3_codes(wi), ref.e4m3_codes(xi)
    ws, xs = np.ones((ref.blocks(n), ref.blocks(k)), np.float32), np.ones((m, ref.blocks(k)), np.float32)
    want = xi.astype(np.float32) @ wi.astype(np.float32).T
    assert np.abs(want).max() <= 256
    wb, wsb, xb, xsb = (GpuBuffer.from_bytes(v.tobytes()) for v in (w, ws, x, xs))
    size = m * n * dt.size_bytes
    out = GpuBuffer.from_bytes(b"\xff" * (size + 64))
    ops.fp8_qmm(dt, wb, wsb, xb, xsb, out, m, n, k)
    raw = out.read_bytes()
    assert raw[size:] == b"\xff" * 64
    assert np.array_equal(unpack_f32(raw[:size], dt).reshape(m, n), want)


@pytest.mark.parametrize("m,n,k", [(1, 200, 400), (40, 300, 272), (300, 300, 400)])
def test_exact_where_sums_are_small_whole_numbers(m, n, k):
    """Codes of small whole numbers and scales of powers of two: every sum is exact, so is the result."""
    rng = np.random.default_rng(m)
    w, x = ref.e4m3_codes(rng.integers(-4, 5, (n, k))), ref.e4m3_codes(rng.integers(-4, 5, (m, k)))
    ws = (2.0 ** rng.integers(-3, 3, (ref.blocks(n), ref.blocks(k)))).astype(np.float32)
    xs = (2.0 ** rng.integers(-3, 3, (m, ref.blocks(k)))).astype(np.float32)
    want = ref.values(x, xs, 1) @ ref.values(w, ws, 128).T
    wb, wsb, xb, xsb = (GpuBuffer.from_bytes(v.tobytes()) for v in (w, ws, x, xs))
    out = GpuBuffer(m * n * 4)
    ops.fp8_qmm(DType.F32, wb, wsb, xb, xsb, out, m, n, k)
    assert np.array_equal(np.frombuffer(out.read_bytes(), "<f4").reshape(m, n), want)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_nan_stays_in_its_row_and_column(m):
    """A NaN code makes its row of x (its row of w) NaN and no other; the rows behind the matrices hold NaN too and reach nothing."""
    n, k = 150, 144
    rng = np.random.default_rng(m)
    w, ws = _weights(rng, n, k)
    x, xs = ref.quantize(rng.standard_normal((m, k)).astype(np.float32), 1)
    w[7, 143] = 127
    if m > 1:
        x[m - 1, 3] = 255
    want = ref.values(x, xs, 1) @ ref.values(w, ws, 128).T
    wb, wsb, xb, xsb = (GpuBuffer.from_bytes(v) for v in (w.tobytes() + b"\x7f" * 65536, ws.tobytes() + b"\xff" * 64, x.tobytes() + b"\x7f" * 65536, xs.tobytes() + b"\xff" * 4096))
    out = GpuBuffer(m * n * 4)
    ops.fp8_qmm(DType.F32, wb, wsb, xb, xsb, out, m, n, k)
    got = np.frombuffer(out.read_bytes(), "<f4").reshape(m, n)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[:, 7]).all()


def test_refusals():
    b = GpuBuffer(1 << 16)
    ok = dict(dt=DType.BF16, w=b, ws=b, x=b, xs=b, out=b, m=2, n=16, k=128)
    for bad in (dict(k=100), dict(k=0), dict(n=0), dict(w=b.ptr + 8), dict(x=b.ptr + 4), dict(w=0), dict(ws=0), dict(x=0), dict(xs=0), dict(out=0), dict(dt=3)):
        a = dict(ok, **bad)
        with pytest.raises(MtqError):
            ops.fp8_qmm(a["dt"], a["w"], a["ws"], a["x"], a["xs"], a["out"], a["m"], a["n"], a["k"])
        if "xs" not in bad:
            with pytest.raises(MtqError):
                ops.fp8_qmv(a["dt"], a["w"], a["ws"], a["x"], a["out"], a["m"], a["n"], a["k"])
    for bad in (dict(cols=24), dict(cols=0), dict(block=2), dict(x=b.ptr + 2), dict(codes=b.ptr + 8), dict(x=0), dict(codes=0), dict(scales=0)):
        a = dict(dict(x=b, codes=b, scales=b, rows=2, cols=128, block=1), **bad)
        with pytest.raises(MtqError):
            ops.fp8_quantize(DType.BF16, a["x"], a["codes"], a["scales"], a["rows"], a["cols"], a["block"])
    ops.fp8_qmm(DType.BF16, b, b, b, b, b, 0, 16, 128)
    ops.fp8_qmv(DType.BF16, b, b, b, b, 0, 16, 128)
    ops.fp8_quantize(DType.BF16, b, b, b, 0, 128, 1)


@pytest.mark.parametrize("m", [1, 3, 16, 40, 300])
def test_captured(m):
    n, k, dt = 400, 656, DType.BF16
    rng = np.random.default_rng(m)
    w, ws = _weights(rng, n, k)
    wb, wsb, xb, out = GpuBuffer.from_bytes(w.tobytes()), GpuBuffer.from_bytes(ws.tobytes()), GpuBuffer(m * k * 2), GpuBuffer(m * n * 2)
    g = Graph()
    try:
        with g:
            ops.fp8_qmv(dt, wb, wsb, xb, out, m, n, k)
        for turn in range(3):
            xb.upload(pack_f32(np.random.default_rng(turn).standard_normal(m * k).astype(np.float32), dt))
            out.upload(b"\xff" * (m * n * 2))
            g.replay()
            first = out.read_bytes()
            ops.fp8_qmv(dt, wb, wsb, xb, out, m, n, k)
            assert out.read_bytes() == first and np.isfinite(unpack_f32(first, dt)).all()
    finally:
        g.close()
