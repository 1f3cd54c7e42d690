"""The operators of an attention layer as a program runs them: three sequences over a paged cache in 4 bits, their prompts and then single tokens.

residual addition, norm and 8 bits -> 8-bit projection to rows of q, k and v -> positions, and keys and values into their pages -> attention -> 8-bit output projection ->
residual addition in place, norm and 8 bits for what comes next. Each stage is held against its definition on what the stage before it left in memory, with that
operator's own bound; nothing waits between the stages while they run. The step of one token a sequence is then captured and replayed, with lengths that grow, against the
same calls made one by one.
"""
import numpy as np
import pytest

from metaltile_amd import GpuBuffer, ops, pack_f32, unpack_f32
from tests import fp8_reference as fp8
from tests import kv_reference as ref
from tests.hip_graph import Graph
from tests.kv_reference import DTYPES, typed
from tests.test_gpu_add_rms_norm_fp8 import EPS, Norm
from tests.test_gpu_fp8 import _tolerance, _weights

pytestmark = pytest.mark.gpu
H, HQ, HKV, DIM, GROUP, PAGE, MOST = 512, 8, 2, 64, 32, 16, 112
WIDTH = (HQ + 2 * HKV) * DIM


class Layer:
    def __init__(self, dt):
        self.dt, self.e = dt, dt.size_bytes
        rng = self.rng = np.random.default_rng(5)
        self.w_in, self.s_in = _weights(rng, WIDTH, H)
        self.w_out, self.s_out = _weights(rng, H, HQ * DIM)
        self.pool = ref.Pool(dt, rng, [90, 20, 50], HKV, DIM, GROUP, PAGE, width=MOST // PAGE).upload()
        angle = np.arange(MOST)[:, None] * 10000.0 ** (-np.arange(0, DIM, 2) / DIM)
        self.table = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
        up = GpuBuffer.from_bytes
        self.b = dict(w_in=up(self.w_in.tobytes()), s_in=up(self.s_in.tobytes()), w_out=up(self.w_out.tobytes()), s_out=up(self.s_out.tobytes()), table=up(self.table.tobytes()))

    def rows(self, rows):
        """Buffers of a call with that many rows a sequence."""
        self.offsets = np.concatenate([[0], np.cumsum(rows)]).astype(int).tolist()
        self.n = n = self.offsets[-1]
        self.first, self.second = Norm(self.dt, n, H, seed=3), Norm(self.dt, n, H, seed=4)
        self.b.update(rows=GpuBuffer(n * WIDTH * self.e), q=GpuBuffer(n * HQ * DIM * self.e), att=GpuBuffer(n * HQ * DIM * self.e))
        self.batch = self.pool.batch(None if len(set(rows)) == 1 else self.offsets, n)

    def inputs(self, lens):
        f = self.first
        f.x, f.r = typed(self.rng.standard_normal((self.n, H)), self.dt), typed(2 * self.rng.standard_normal((self.n, H)), self.dt)
        f.xb.upload(pack_f32(f.x, self.dt))
        f.rb.upload(pack_f32(f.r, self.dt))
        self.pool.lens = list(lens)
        self.pool.lb.upload(np.array(lens, "<u4").tobytes())

    def run(self):
        b, dt, n, f, s = self.b, self.dt, self.n, self.first, self.second
        f.call()
        ops.fp8_qmm(dt, b["w_in"], b["s_in"], f.codes, f.scales, b["rows"], n, WIDTH, H)
        k = b["rows"].ptr + HQ * DIM * self.e
        ops.kv_append(dt, self.pool.cache, self.batch, k, k + HKV * DIM * self.e, row_stride=(WIDTH, WIDTH, WIDTH), q=b["rows"], q_out=b["q"], hq=HQ, cos_sin=b["table"], n_positions=MOST, rot=DIM)
        ops.kv_attention(dt, self.pool.cache, self.batch, b["q"], b["att"], HQ, DIM ** -0.5)
        ops.fp8_qmv(dt, b["w_out"], b["s_out"], b["att"], s.xb, n, H, HQ * DIM)
        ops.add_rms_norm_fp8(dt, s.xb, f.sum, s.wb, EPS, f.sum, s.codes, s.scales, n, H)

    def outputs(self):
        f, s = self.first, self.second
        return [x.read_bytes() for x in (f.codes, f.scales, f.sum, self.b["rows"], self.b["q"], self.b["att"], s.xb, s.codes, s.scales, *self.pool.bufs)]

    def hold(self):
        b, dt, n, f, s, pool = self.b, self.dt, self.n, self.first, self.second, self.pool
        typed_of = lambda buf, *shape: unpack_f32(buf.read_bytes(), dt).reshape(shape)
        f.hold(sum_buf=None)
        rows = typed_of(b["rows"], n, HQ + 2 * HKV, DIM)
        xv, wv = fp8.values(*f.outputs(), 1), fp8.values(self.w_in, self.s_in, 128)
        want = xv @ wv.T
        assert np.all(np.abs(rows.reshape(n, -1) - want) <= _tolerance(xv, wv, want, dt, H))
        q = typed_of(b["q"], n, HQ, DIM)
        for seq, row, place in ref.spans(pool.lens, self.offsets, pool.max_len):
            at = np.array([place])
            assert np.array_equal(q[row], typed(ref.turned(rows[row:row + 1, :HQ], at, self.table, DIM, False), dt)[0])
            page = pool.pages[seq, place // PAGE]
            for part, x in zip(pool.parts, (ref.turned(rows[row:row + 1, HQ:HQ + HKV], at, self.table, DIM, False), rows[row:row + 1, HQ + HKV:])):
                for arr, new in zip(part, ref.quantize(x[0], GROUP, dt)):
                    arr[page, :, place % PAGE] = new
        for got, want in zip(pool.downloaded(), pool.parts):
            assert all(np.array_equal(x, y, equal_nan=True) for x, y in zip(got, want))
        att = typed_of(b["att"], n, HQ, DIM)
        many = dt.size_bytes == 2 and n * HQ // HKV > 64 * len(pool.lens)
        want, tol = ref.attention(pool, q, self.offsets, HQ, DIM ** -0.5, 0, dt, rounded=many)
        assert np.all(np.abs(att - want) <= tol)
        y = typed_of(s.xb, n, H)
        xv, wv = fp8.values(*fp8.quantize(att.reshape(n, -1), 1), 1), fp8.values(self.w_out, self.s_out, 128)
        want = xv @ wv.T
        assert np.all(np.abs(y - want) <= _tolerance(xv, wv, want, dt, HQ * DIM))
        s.x, s.r = y, typed((f.x + f.r).astype(np.float32), dt)
        s.hold(sum_buf=f.sum)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_prompt_and_tokens(dt):
    print(f"[case] kv layer {dt.name}", flush=True)
    layer = Layer(dt)
    lens = [70, 1, 33]
    layer.rows(lens)
    layer.inputs(lens)
    layer.run()
    layer.hold()
    layer.rows([1, 1, 1])
    g = None
    try:
        for turn in range(5):
            lens = [n + 1 for n in lens]
            layer.inputs(lens)
            if g is None:
                layer.run()
                layer.hold()
                g = Graph()
                with g:
                    layer.run()
                continue
            g.replay()
            layer.hold()
            replayed = layer.outputs()
            layer.run()
            ops.sync()
            assert layer.outputs() == replayed
    finally:
        if g is not None:
            g.close()


@pytest.mark.parametrize("kernel", [1, 4])
def test_two_captured_graphs(kernel):
    """Two captured layers that share the library's buffers, replayed in turn, and the buffers of calls between them that want more."""
    from metaltile_amd import DType, _lib
    from metaltile_amd.runtime import _ensure_init
    lib = _ensure_init()
    _lib.check(lib.mtq_set_option(b"kv.kernel", kernel))
    _lib.check(lib.mtq_set_option(b"kv.slices", 3))
    graphs = []
    try:
        layers = [Layer(dt) for dt in (DType.BF16, DType.F16)]
        for layer, rows in zip(layers, ([20, 1, 7], [2, 2, 2])):
            layer.rows(rows)
            layer.inputs([70, 1, 33] if rows[1] == 1 else [60, 2, 40])
            layer.run()
            ops.sync()
            graphs.append(Graph())
            with graphs[-1]:
                layer.run()
        want = []
        for layer in layers:
            layer.run()
            ops.sync()
            want.append(layer.outputs())
        from tests.test_gpu_kv_attention import Attention
        between = Attention(DType.BF16, [1500, 300], [40, 30], hq=16, hkv=2)
        for turn in range(3):
            for g in graphs:
                g.replay()
            between.call()
            for g in reversed(graphs):
                g.replay()
            ops.sync()
            assert [layer.outputs() for layer in layers] == want
            between.hold(kernel)
    finally:
        for g in graphs:
            g.close()
        for name in (b"kv.kernel", b"kv.slices"):
            _lib.check(lib.mtq_set_option(name, 0))
