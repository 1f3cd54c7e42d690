"""Log probabilities, entropy and top alternatives of rows of logits, against 64 bits.

Tolerance. With d = x - m (one rounding), e = exp(d) and z, s sums of n positive terms: a term is off by the rounding of d log2(e) in the
exponent, |d| 2^-24 (with e^d |d| <= 1 / e: at most 2^-24 of z in all for every further term of that size), and by an ulp of the hardware's
exponential, 2^-23; a lane adds 32 elements of a tile, then tiles, then lanes, waves and slices, less than 128 additions in a row, 2^-24 each.
So z and s are off by less than 160 x 2^-24 < 1e-5 of themselves, log z by that, and a difference x - m - log z by another 2^-23 of the
larger of its parts: 1e-5 + 2^-22 max(|x - m|, log z) for a log probability, 1e-5 (1 + log z + |s / z|) for the entropy.
"""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests.hip_graph import Graph

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]
UNTOUCHED = 0x7FC12345   # a NaN of its own


def _reference(x, tokens, k):
    """x f64 [rows, vocab] of values of the element type."""
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        m = np.where(np.isfinite(m), m, np.where(np.isnan(m) | (m > 0), np.nan, 0.0))
        d = x - m
        e = np.where(np.isnan(d), np.nan, np.exp(d))
        z = e.sum(1, keepdims=True)
        s = np.where(e == 0, 0.0, e * np.where(e == 0, 0.0, d)).sum(1, keepdims=True)
        lp = np.where(z == 0, -np.inf, d - np.log(z))
        entropy = np.where(z == 0, 0.0, np.log(z) - s / z)[:, 0]
        size = 1 + np.abs(np.log(np.where(z == 0, 1, z))) + np.abs(np.where(z == 0, 0, s / z))
    order = np.where(np.isnan(x), -np.inf, x)
    ids = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), np.isnan(x), -order), axis=1)[:, :k]
    out = np.take_along_axis(np.isnan(x), ids, 1)
    return np.take_along_axis(lp, tokens, 1), entropy, np.where(out, 0xFFFFFFFF, ids), np.where(out, np.nan, np.take_along_axis(lp, ids, 1)), size[:, 0], d, z


def _close(got, want, tol):
    with np.errstate(all="ignore"):
        want = np.asarray(want, np.float64).astype(np.float32).astype(np.float64)   # (a difference past the f32 range is -inf)
        same = (np.isnan(got) & np.isnan(want)) | (got == want)
        return bool(np.all(same | (np.abs(got - want) <= tol)))


def _call(dt, x, tokens, k, pad=0, shift=0, want_entropy=True):
    """x f32 [rows, vocab] -> (values of x in the type, outputs). Rows begin `shift` elements into a buffer, vocab + pad apart; between them are NaNs."""
    rows, vocab = x.shape
    buf = np.full((rows, vocab + pad), np.nan, np.float32)
    buf[:, :vocab] = x
    flat = np.concatenate([np.full(shift, np.nan, np.float32), buf.reshape(-1)])
    logits = GpuBuffer.from_bytes(pack_f32(flat, dt))
    given = GpuBuffer.from_bytes(tokens.astype("<u4").tobytes())
    fill = lambda n: GpuBuffer.from_bytes(np.full(max(n, 1), UNTOUCHED, "<u4").tobytes())
    outs = lp, ent, ids, top = [fill(n) for n in (tokens.size, rows, rows * k, rows * k)]
    call = lambda: ops.token_logprobs(dt, logits.ptr + shift * dt.size_bytes, vocab + pad, given, tokens.shape[1], lp, ent if want_entropy else None, ids, top, k, rows, vocab)
    call()
    read = lambda: (np.frombuffer(lp.read_bytes(4 * tokens.size), "<f4").reshape(tokens.shape), np.frombuffer(ent.read_bytes(4 * rows), "<f4"),
                    np.frombuffer(ids.read_bytes(4 * rows * k) if k else b"", "<u4").reshape(rows, k),
                    np.frombuffer(top.read_bytes(4 * rows * k) if k else b"", "<f4").reshape(rows, k))
    values = unpack_f32(pack_f32(x, dt), dt).reshape(x.shape).astype(np.float64)
    return values, read, call, [logits, given, *outs]


def _hold(values, tokens, k, got):
    lp, ent, ids, top = got
    safe = np.minimum(tokens, values.shape[1] - 1).astype(np.int64)
    want = _reference(values, safe, k)
    with np.errstate(all="ignore"):
        tol = 1e-5 + 2.0 ** -22 * np.maximum(np.nanmax(np.where(np.isfinite(want[5]), np.abs(want[5]), 0), 1, initial=0), np.nan_to_num(np.abs(np.log(want[6][:, 0])), posinf=0, neginf=0))
    there = tokens < values.shape[1]
    assert _close(np.where(there, lp, 0), np.where(there, want[0], 0), tol[:, None])
    assert np.all(lp.view("<u4")[~there] == UNTOUCHED)
    assert _close(ent, want[1], 1e-5 * want[4])
    assert np.array_equal(ids, want[2])
    assert _close(top, want[3], tol[:, None])


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,vocab,k,given,pad,shift", [
    (1, 1, 1, 1, 0, 0), (1, 1, 0, 1, 0, 3), (3, 2, 2, 2, 5, 1), (2, 31, 31, 1, 0, 1), (5, 64, 32, 3, 1, 0), (1, 2047, 5, 1, 0, 7), (1, 2048, 5, 1, 0, 0), (1, 2049, 20, 1, 0, 0),
    (4, 8191, 32, 70, 2, 5), (2, 8193, 1, 1, 0, 0), (1, 32000, 8, 1, 0, 0), (7, 50257, 20, 1, 47, 0), (1, 128256, 32, 2, 0, 3), (33, 9001, 5, 1, 3, 1), (1030, 300, 5, 1, 0, 0),
    (1100, 4099, 3, 1, 1, 1), (2, 262147, 17, 1, 0, 0)])
def test_against_64_bits(dt, rows, vocab, k, given, pad, shift):
    print(f"[case] token_logprobs {dt.name} rows{rows} vocab{vocab} k{k} given{given} pad{pad} shift{shift}", flush=True)
    rng = np.random.default_rng(rows + vocab + k)
    x = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    tokens = rng.integers(0, vocab, (rows, given))
    tokens[0, 0] = 0xFFFFFFFF if given > 1 else vocab - 1
    values, read, _, bufs = _call(dt, x, tokens, k, pad, shift)
    _hold(values, tokens, k, read())
    for b in bufs:
        b.free()


KINDS = ["equal", "ascending", "descending", "one_left", "half_masked", "all_masked", "lowest", "huge", "nan", "all_nan", "plus_inf", "zeros_of_both_signs", "peaked", "last_only"]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab,k", [(2, 700, 32), (1, 20000, 20), (1025, 513, 5)])
def test_rows_of_their_own(dt, kind, rows, vocab, k):
    print(f"[case] token_logprobs {dt.name} {kind} rows{rows} vocab{vocab} k{k}", flush=True)
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    low = {DType.F32: np.float32(-3.4028235e38), DType.F16: np.float32(-65504), DType.BF16: np.float32(-3.3895314e38)}[dt]
    if kind == "equal": x[:] = 1.25
    elif kind == "ascending": x = np.sort(x, 1)
    elif kind == "descending": x = -np.sort(-x, 1)
    elif kind == "one_left": x[:, np.arange(vocab) != vocab // 3] = -np.inf
    elif kind == "half_masked": x[:, :vocab // 2] = -np.inf
    elif kind == "all_masked": x[:] = -np.inf
    elif kind == "lowest": x[:, 3:] = low
    elif kind == "huge": x[:, ::2] = -low * np.float32(0.5); x[:, 1::2] = low
    elif kind == "nan": x[0, vocab - 5] = np.nan; x[-1, 2] = -np.inf
    elif kind == "all_nan": x[0] = np.nan
    elif kind == "plus_inf": x[0, 5] = np.inf; x[0, 77] = np.inf
    elif kind == "zeros_of_both_signs": x[:] = 0.0; x[:, ::3] = -0.0
    elif kind == "peaked": x[:, 17] = 60.0
    elif kind == "last_only": x[:] = -np.inf; x[:, -1] = -3.0
    tokens = rng.integers(0, vocab, (rows, 2))
    values, read, _, bufs = _call(dt, x, tokens, k)
    _hold(values, tokens, k, read())
    for b in bufs:
        b.free()


def test_outputs_that_are_not_wanted():
    lib = _ensure_init()
    x = np.random.default_rng(5).standard_normal((3, 5000)).astype(np.float32)
    logits, toks, out = GpuBuffer.from_bytes(x.tobytes()), GpuBuffer.from_bytes(np.arange(3, dtype="<u4").tobytes()), GpuBuffer.from_bytes(bytes(3 * 4 * 4))
    ops.token_logprobs(DType.F32, logits, 5000, toks, 1, out, None, None, None, 4, 3, 5000)
    want = _reference(x.astype(np.float64), np.arange(3)[:, None], 4)
    assert _close(np.frombuffer(out.read_bytes(12), "<f4"), want[0][:, 0], 2e-5)
    ops.token_logprobs(DType.F32, logits, 5000, None, 0, None, out, None, None, 0, 3, 5000)
    assert _close(np.frombuffer(out.read_bytes(12), "<f4"), want[1], 2e-4)
    ops.token_logprobs(DType.F32, logits, 5000, None, 0, None, None, out, None, 4, 3, 5000)
    assert np.array_equal(np.frombuffer(out.read_bytes(48), "<u4").reshape(3, 4), want[2])
    ops.token_logprobs(DType.F32, logits, 5000, None, 0, None, None, None, out, 4, 3, 5000)
    assert _close(np.frombuffer(out.read_bytes(48), "<f4").reshape(3, 4), want[3], 2e-5)
    ops.token_logprobs(DType.F32, logits, 5000, None, 0, None, None, None, None, 4, 3, 5000)
    for bad in (dict(tokens=None), dict(lp=None), dict(logits=0), dict(logits=logits.ptr + 2), dict(stride=4999), dict(top=33)):
        a = dict(dict(logits=logits.ptr, tokens=toks, lp=out, stride=5000, top=1), **bad)
        with pytest.raises(MtqError):
            ops.token_logprobs(DType.F32, a["logits"], a["stride"], a["tokens"], 1, a["lp"], None, None, None, a["top"], 3, 5000) if a["top"] == 1 else \
                ops.token_logprobs(DType.F32, a["logits"], a["stride"], a["tokens"], 1, a["lp"], None, out, None, a["top"], 3, 5000)
    # without memory for the slices a workgroup has a row to itself: the same values
    _lib.check(lib.mtq_set_option(b"scratch.most_kb", 1))
    try:
        one = np.random.default_rng(6).standard_normal((1, 90000)).astype(np.float32)
        values, read, _, bufs = _call(DType.F32, one, np.array([[11]]), 20)
        _hold(values, np.array([[11]]), 20, read())
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))


def test_captured():
    rng = np.random.default_rng(8)
    x = (2.5 * rng.standard_normal((2, 40000))).astype(np.float32)
    tokens = rng.integers(0, 40000, (2, 1))
    g = Graph()
    try:
        values, read, call, bufs = _call(DType.BF16, x, tokens, 20)
        with g:
            call()
        for turn in range(3):
            y = (2.5 * np.random.default_rng(turn).standard_normal((2, 40000))).astype(np.float32)
            bufs[0].upload(pack_f32(y, DType.BF16))
            g.replay()
            replayed = [v.copy() for v in read()]
            _hold(unpack_f32(pack_f32(y, DType.BF16), DType.BF16).reshape(2, -1).astype(np.float64), tokens, 20, replayed)
            call()   # the program's own call between replays, through the same buffer
            assert all(np.array_equal(a.view("<u4"), b.view("<u4")) for a, b in zip(replayed, read()))
    finally:
        g.close()
