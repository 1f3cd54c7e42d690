"""The served operators where sizes, sharing and order are at their edges: offsets past 32 bits, scratch that grows behind a captured graph, calls one
behind the other, many sequences, streams of the caller's.
"""
import ctypes as C

import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests import fp8_reference as ref
from tests.hip_graph import Graph
from tests.test_gpu_fp8 import _tolerance, _weights
from tests.test_gpu_gated_delta import Case, rule
from tests.test_gpu_token_logprobs import _close, _reference

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]


def _put(buf, at, data):
    arr = np.frombuffer(data, np.uint8)
    assert at + arr.nbytes <= buf.nbytes
    _lib.check(_ensure_init().mtq_upload(buf.ptr + at, arr.ctypes.data_as(C.c_void_p), arr.nbytes))


def _get(buf, at, dtype, count):
    out = np.empty(count, dtype)
    assert at + out.nbytes <= buf.nbytes
    _lib.check(_ensure_init().mtq_download(out.ctypes.data_as(C.c_void_p), buf.ptr + at, out.nbytes))
    return out


# ---- many chunks, sequences and heads

MANY = [  # lens, hk, hv, dk, dv: one workgroup for a key head's value heads, more than four of these, more sequences than a wave has lanes, more walks than CUs
    ([4480], 8, 16, 64, 16), ([260] * 64, 2, 12, 32, 16), ([(7 * i) % 5 * 40 + i % 3 for i in range(150)], 2, 4, 64, 32), ([0] * 70 + [100, 0, 33] + [1] * 70 + [65], 1, 2, 128, 16),
    ([90, 70, 33, 1, 17] * 8, 1, 4, 64, 80), ([130] * 20, 4, 8, 128, 64)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,hk,hv,dk,dv", MANY, ids=lambda v: str(v).replace(" ", "")[:40])
def test_delta_many(dt, lens, hk, hv, dk, dv):
    print(f"[case] gated_delta_rule {dt.name} {len(lens)} sequences of {sum(lens)} tokens hk{hk} hv{hv} dk{dk} dv{dv}", flush=True)
    c = Case(dt, lens, hk, hv, dk, dv)
    c.call()
    c.hold()


def test_delta_slots_of_a_large_pool():
    """States past 2^32 elements: only the named slots are written."""
    hk, hv, dk, dv, n_slots = 2, 32, 128, 128, 8300
    one = hv * dv * dk
    assert (n_slots - 1) * one > 1 << 32
    for lens in ([1, 1], [40, 70]):
        c = Case(DType.BF16, lens, hk, hv, dk, dv, slots=[8299, 3], n_slots=1)   # (its own states are not used)
        pool = GpuBuffer(n_slots * one * 4)
        rng = np.random.default_rng(5)
        states = (0.3 * rng.standard_normal((2, hv, dv, dk))).astype(np.float32)
        for slot, s in zip(c.slots, states):
            _put(pool, slot * one * 4, s.tobytes())
        _put(pool, 8298 * one * 4, np.full(one, 5.5, "<f4").tobytes())
        ops.gated_delta_rule(c.dt, *c.at, c.gb, c.bb, pool, pool, c.y, 2, c.tokens, hk, hv, dk, dv, row_stride=c.strides, offsets=c.ob, slots=c.sb, n_slots=n_slots, scale=c.scale, norm_eps=c.eps)
        far = [_get(pool, slot * one * 4, "<f4", one) for slot in c.slots]
        y = c.y.read_bytes()
        assert np.all(_get(pool, 8298 * one * 4, "<f4", one) == 5.5)
        pool.free()
        near = Case(DType.BF16, lens, hk, hv, dk, dv)
        near.state = states
        near.state_in.upload(states.tobytes())
        near.call()
        near.hold()
        assert y == near.y.read_bytes()
        assert np.array_equal(np.stack(far).reshape(states.shape), near.results()[1])


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=str)
@pytest.mark.parametrize("most_kb", [0, 400])
def test_delta_no_numbers(dt, what, bad, most_kb):
    """A NaN or an infinity reaches what comes behind it in its sequence, its head and, from v and the state, its column, and nothing else: not the tokens
    before it, of the same chunk or others, in prompts, short sequences and single tokens, with all chunks at once or in windows."""
    lens, hk, hv, dk, dv = [150, 5, 200, 1, 70, 64], 2, 4, 64, 48
    c = Case(dt, lens, hk, hv, dk, dv)
    at = {"q": (c.q, [(70, 1, 3), (352, 0, 0), (375, 0, 5)]), "k": (c.k, [(70, 1, 3), (152, 0, 0), (300, 0, 9)]), "v": (c.v, [(70, 1, 3), (153, 2, 5), (300, 0, 40), (420, 3, 47), (489, 0, 0)]),
          "g": (c.g, [(70, 1), (152, 0), (300, 3)]), "beta": (c.beta, [(70, 1), (152, 0), (300, 3), (355, 2)]), "state": (c.state, [(0, 1, 3, 5), (2, 0, 0, 0), (3, 2, 40, 63)])}[what]
    for i in at[1]:
        at[0][i] = bad
    c.bufs[0].upload(pack_f32(np.concatenate([x.reshape(c.tokens, -1) for x in (c.q, c.k, c.v)], 1).astype(np.float32), dt))
    c.gb.upload(c.g.tobytes())
    c.bb.upload(c.beta.tobytes())
    c.state_in.upload(c.state.tobytes())
    lib = _ensure_init()
    try:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", most_kb))
        c.call()
        y, S = c.results()
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
    with np.errstate(all="ignore"):
        wy, wS = rule(*(x.astype(np.float64) for x in (c.q, c.k, c.v, c.g, c.beta, c.state)), list(zip(c.offsets[:-1], c.offsets[1:])), range(len(lens)), c.scale, c.eps)
        assert np.array_equal(np.isfinite(y), np.isfinite(wy)) and np.array_equal(np.isfinite(S), np.isfinite(wS))
        assert not np.isfinite(y).all() and np.isfinite(y).mean() > 0.5
        rel = (dk / 16 + 16) * 2.0 ** -24 * 200
        for got, want in ((y, wy), (S, wS)):
            fine = np.isfinite(want)
            assert np.all(np.abs(got[fine] - want[fine]) <= rel * np.abs(want[fine]).max())


# ---- offsets past 32 bits

@pytest.mark.parametrize("rows", [3, 300])
def test_logprobs_far_rows(rows):
    vocab, k = 1000, 4
    stride = ((1 << 32) // (rows - 1) // 8 + 1) * 8
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((1, vocab)).astype(np.float32)
    logits = GpuBuffer(((rows - 1) * stride + vocab) * 2)
    _put(logits, (rows - 1) * stride * 2, pack_f32(x, DType.BF16))
    given = GpuBuffer.from_bytes(np.full(rows, 17, "<u4").tobytes())
    lp, ent, ids, top = (GpuBuffer(4 * n) for n in (rows, rows, rows * k, rows * k))
    ops.token_logprobs(DType.BF16, logits, stride, given, 1, lp, ent, ids, top, k, rows, vocab)
    xv = unpack_f32(pack_f32(x, DType.BF16), DType.BF16).reshape(1, vocab).astype(np.float64)
    wlp, went, wids, wtop, size, d, z = _reference(xv, np.array([[17]]), k)
    tol = 1e-5 + 2.0 ** -22 * 10
    assert _close(_get(lp, 4 * (rows - 1), "<f4", 1), wlp[0], tol) and _close(_get(ent, 4 * (rows - 1), "<f4", 1), went, 1e-5 * size)
    assert np.array_equal(_get(ids, 4 * (rows - 1) * k, "<u4", k), wids[0]) and _close(_get(top, 4 * (rows - 1) * k, "<f4", k), wtop[0], tol)


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_far_rows(block):
    rows, cols = 65540, 65552
    x = GpuBuffer(rows * cols * 2)
    rng = np.random.default_rng(block)
    last = unpack_f32(pack_f32(rng.standard_normal((4, cols)).astype(np.float32), DType.BF16), DType.BF16).reshape(4, cols)   # the last block's only rows
    _put(x, (rows - 4) * cols * 2, pack_f32(last, DType.BF16))
    codes, scales = GpuBuffer(rows * cols), GpuBuffer(4 * -(-rows // block) * ref.blocks(cols))
    ops.fp8_quantize(DType.BF16, x, codes, scales, rows, cols, block)
    wc, ws = ref.quantize(last, block)
    assert np.array_equal(_get(codes, (rows - 4) * cols, np.uint8, 4 * cols).reshape(4, cols), wc)
    n = ws.size
    assert np.array_equal(_get(scales, scales.nbytes - 4 * n, "<f4", n).reshape(ws.shape), ws)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_product_far_weights(m):
    """Rows of w past 4 GiB; before them is whatever the memory held."""
    n, k, dt, tail = 66000, 65552, DType.F32, 80          # (the last rows are a block of 128 rows of their own: 66000 = 515 x 128 + 80)
    rng = np.random.default_rng(m)
    wt, wst = _weights(rng, tail, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    codes, scales = ref.quantize(x, 1)
    w, ws = GpuBuffer(n * k), GpuBuffer(4 * ref.blocks(n) * ref.blocks(k))
    _put(w, (n - tail) * k, wt.tobytes())
    _put(ws, ws.nbytes - wst.nbytes, wst.tobytes())
    xb, out = GpuBuffer.from_bytes(x.tobytes()), GpuBuffer(4 * m * n)
    ops.fp8_qmv(dt, w, ws, xb, out, m, n, k)
    got = np.frombuffer(out.read_bytes(), "<f4").reshape(m, n)[:, n - tail:].astype(np.float64)
    xv, wv = ref.values(codes, scales, 1), ref.values(wt, wst, 128)
    want = xv @ wv.T
    assert np.all(np.abs(got - want) <= _tolerance(xv, wv, want, dt, k))


def test_product_far_rows_and_results():
    """Results past 2^32 bytes and rows of x past 2^32 bytes, in tiles."""
    m, n, k, dt, tail = 600000, 4096, 16384, DType.BF16, 40
    rng = np.random.default_rng(1)
    w, ws = _weights(rng, n, k)
    xt, xst = ref.quantize(rng.standard_normal((tail, k)).astype(np.float32), 1)
    wb, wsb = GpuBuffer.from_bytes(w.tobytes()), GpuBuffer.from_bytes(ws.tobytes())
    x, xs, out = GpuBuffer(m * k), GpuBuffer(4 * m * ref.blocks(k)), GpuBuffer(2 * m * n)
    _put(x, (m - tail) * k, xt.tobytes())
    _put(xs, 4 * (m - tail) * ref.blocks(k), xst.tobytes())
    ops.fp8_qmm(dt, wb, wsb, x, xs, out, m, n, k)
    got = unpack_f32(_get(out, 2 * (m - tail) * n, np.uint8, 2 * tail * n).tobytes(), dt).reshape(tail, n).astype(np.float64)
    xv, wv = ref.values(xt, xst, 1), ref.values(w, ws, 128)
    want = xv @ wv.T
    assert np.all(np.abs(got - want) <= _tolerance(xv, wv, want, dt, k))


# ---- scratch and streams

class _Product:
    def __init__(self, m, n, k, seed):
        rng = np.random.default_rng(seed)
        self.shape = m, n, k
        w, ws = _weights(rng, n, k)
        self.w, self.ws = GpuBuffer.from_bytes(w.tobytes()), GpuBuffer.from_bytes(ws.tobytes())
        self.x = GpuBuffer.from_bytes(pack_f32(rng.standard_normal((m, k)).astype(np.float32), DType.BF16))
        self.out = GpuBuffer(2 * m * n)

    def call(self):
        ops.fp8_qmv(DType.BF16, self.w, self.ws, self.x, self.out, *self.shape)


def test_calls_one_behind_the_other_share_scratch():
    """No wait between them: each uses the scratch that the one before may still have."""
    delta, small, large = Case(DType.F16, [300, 1, 90], 2, 4, 64, 64), _Product(8, 300, 512, 1), _Product(500, 700, 1024, 2)
    rng = np.random.default_rng(3)
    x = GpuBuffer.from_bytes(rng.standard_normal((3, 70000)).astype(np.float32).tobytes())
    ids, top = GpuBuffer(4 * 3 * 8), GpuBuffer(4 * 3 * 8)
    logprobs = lambda: ops.token_logprobs(DType.F32, x, 70000, None, 0, None, None, ids, top, 8, 3, 70000)
    calls, outs = [delta.call, small.call, large.call, logprobs], [delta.y, delta.state_out, small.out, large.out, ids, top]
    for c in calls:
        c()
        ops.sync()
    want = [b.read_bytes() for b in outs]
    for order in ([0, 1, 2, 3], [3, 2, 1, 0], [1, 0, 3, 2], [2, 3, 0, 1]):
        for b in outs:
            b.zero()
        for i in order * 2:
            calls[i]()
        assert [b.read_bytes() for b in outs] == want, order


def test_scratch_that_grows_behind_a_graph():
    """Two graphs captured around a call that needs more scratch, replayed among eager calls that use it."""
    a, b, large, huge = _Product(8, 300, 512, 1), Case(DType.BF16, [200, 90], 2, 4, 128, 64), _Product(700, 500, 2048, 2), Case(DType.BF16, [3000, 2000], 2, 4, 128, 64)
    for c in (a, b):
        c.call()
    want = a.out.read_bytes(), b.y.read_bytes(), b.state_out.read_bytes()
    first, second = Graph(), None
    try:
        with first:
            a.call()
            b.call()
        large.call()
        second = Graph()   # (waits for the stream that is left)
        with second:
            b.call()
            a.call()
        huge.call()
        ops.sync()
        for turn in range(3):
            for g in (first, second):
                for buf in (a.out, b.y, b.state_out):
                    buf.zero()
                ops.sync()   # (the graphs have streams of their own)
                g.replay()
                assert (a.out.read_bytes(), b.y.read_bytes(), b.state_out.read_bytes()) == want
                (large, huge)[turn % 2].call()
                ops.sync()
    finally:
        if second is not None:
            second.close()
        first.close()


def test_without_scratch():
    """No room for the slices of few rows: a workgroup has each row. Activations that go through scratch are an error; a single row does not."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 50000)).astype(np.float32)
    logits, given = GpuBuffer.from_bytes(x.tobytes()), GpuBuffer.from_bytes(np.array([5, 49999], "<u4").tobytes())
    lp, ent, ids, top = (GpuBuffer(4 * n) for n in (2, 2, 10, 10))
    several, single = _Product(40, 300, 512, 1), _Product(1, 300, 512, 1)
    single.call()
    want = single.out.read_bytes()
    lib = _ensure_init()
    try:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 1))
        ops.token_logprobs(DType.F32, logits, 50000, given, 1, lp, ent, ids, top, 5, 2, 50000)
        with pytest.raises(MtqError):
            several.call()
        single.out.zero()
        single.call()
        assert single.out.read_bytes() == want
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
    wlp, went, wids, wtop, size, d, z = _reference(x.astype(np.float64), np.array([[5], [49999]]), 5)
    read = lambda b, *shape: np.frombuffer(b.read_bytes(), "<f4").reshape(shape)
    tol = 1e-5 + 2.0 ** -22 * 20
    assert _close(read(lp, 2, 1), wlp, tol) and _close(read(ent, 2), went, 1e-5 * size) and _close(read(top, 2, 5), wtop, tol)
    assert np.array_equal(np.frombuffer(ids.read_bytes(), "<u4").reshape(2, 5), wids)


def test_streams_of_the_callers():
    """From the library's own stream to two of the caller's."""
    lib, hip = _ensure_init(), C.CDLL("libamdhip64.so")
    hip.hipStreamCreate.argtypes, hip.hipStreamDestroy.argtypes = [C.POINTER(C.c_void_p)], [C.c_void_p]
    delta, product = Case(DType.F32, [150, 40], 1, 2, 64, 64), _Product(40, 300, 512, 1)
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        assert hip.hipStreamCreate(C.byref(s)) == 0
    try:
        got = []
        for s in (None, *streams):
            _lib.check(lib.mtq_set_stream(s))
            for b in (delta.y, delta.state_out, product.out):
                b.zero()
            delta.call()
            product.call()
            ops.sync()
            got.append([b.read_bytes() for b in (delta.y, delta.state_out, product.out)])
        assert got[0] == got[1] == got[2]
    finally:
        _lib.check(lib.mtq_sync())
        _lib.check(lib.mtq_set_stream(None))
        for s in streams:
            assert hip.hipStreamDestroy(s) == 0


def test_misaligned_buffers_are_refused():
    """Every pointer in turn off its type's alignment: an error before any launch."""
    b = GpuBuffer(1 << 16)
    p = b.ptr
    def refused(call, args, off):
        call(*args)   # (as they are: fine)
        for i, by in off:
            bad = list(args)
            bad[i] += by
            with pytest.raises(MtqError):
                call(*bad)
    # (one zero-filled buffer stands for all arguments: results land where nothing reads them, ids are 0)
    o = p + (1 << 15)
    refused(lambda x, c, s: ops.fp8_quantize(DType.BF16, x, c, s, 2, 64, 1), (p, o, o + 4096), ((0, 2), (0, 8), (1, 4), (2, 2)))
    refused(lambda w, ws, x, xs, out: ops.fp8_qmm(DType.BF16, w, ws, x, xs, out, 2, 16, 64), (p, p + 4096, p, p + 4096, o), ((0, 8), (1, 2), (2, 8), (3, 2), (4, 1)))
    refused(lambda w, ws, x, out: ops.fp8_qmv(DType.F32, w, ws, x, out, 1, 16, 64), (p, p + 4096, p, o), ((0, 8), (1, 2), (2, 8), (3, 2)))
    refused(lambda q, k, v, g, beta, si, so, y: ops.gated_delta_rule(DType.F16, q, k, v, g, beta, si, so, y, 1, 2, 1, 1, 16, 16), (p, p, p, p, p, p + 4096, o, o + 8192),
            ((0, 1), (1, 1), (2, 1), (3, 2), (4, 2), (5, 2), (6, 2), (7, 2)))
    refused(lambda x, t, lp, e, ids, top: ops.token_logprobs(DType.BF16, x, 64, t, 1, lp, e, ids, top, 2, 1, 64), (p, p, o, o + 64, o + 128, o + 256),
            ((0, 1), (1, 2), (2, 2), (3, 2), (4, 2), (5, 2)))
    ops.sync()
