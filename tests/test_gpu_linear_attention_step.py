"""The served operators as a program runs them: a linear-attention layer and a head over three sequences, a prompt and then single tokens.

x -> 8-bit projection to rows of q, k, v and z -> gated delta rule over the sequences' states -> gated RMS norm and 4-bit output projection (a call
for each sequence) -> 8-bit head -> log probabilities and likeliest tokens. Each stage is held against 64 bits on what the stage before it left
in memory, with that operator's own bound; nothing waits between the stages while they run. The step of one token a sequence is then captured
and replayed, the states carried on in place, against the same calls made one by one.
"""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, ops, pack_f32, unpack_f32
from metaltile_amd.synth import make_case
from tests import fp8_reference as ref
from tests.hip_graph import Graph
from tests.parity import rel_err
from tests.test_gpu_fp8 import _tolerance, _weights
from tests.test_gpu_gated_delta import rule
from tests.test_gpu_gated_rms_norm_qmv import ODT, TOL
from tests.test_gpu_token_logprobs import _close, _reference

pytestmark = pytest.mark.gpu
H, HK, HV, DK, DV, VOCAB, TOP, SLOTS, EPS = 512, 2, 4, 64, 64, 1000, 4, 6, 1e-6
WIDTH = 2 * HK * DK + 2 * HV * DV   # q, k, v, z


class Layer:
    def __init__(self, oracle, dt):
        self.oracle, self.dt, self.e = oracle, dt, dt.size_bytes
        rng = self.rng = np.random.default_rng(11)
        self.w_in, self.s_in = _weights(rng, WIDTH, H)
        self.w_head, self.s_head = _weights(rng, VOCAB, H)
        self.c = make_case(31, dt, 4, 64, 1, H, HV * DV, bias_rule="midpoint")
        self.nw = oracle.round_through((1 + 0.2 * rng.standard_normal(DV)).astype(np.float32), ODT[dt])
        self.slots = [4, 0, 2]
        state = (0.1 * rng.standard_normal((SLOTS, HV, DV, DK))).astype(np.float32)
        up = GpuBuffer.from_bytes
        self.b = {k: up(v) for k, v in dict(w_in=self.w_in.tobytes(), s_in=self.s_in.tobytes(), w_head=self.w_head.tobytes(), s_head=self.s_head.tobytes(), w4=self.c.w.tobytes(),
                                            s4=self.c.scales_bytes, b4=self.c.biases_bytes, nw=pack_f32(self.nw, dt), eps=np.float32(EPS).tobytes(),
                                            slots=np.array(self.slots, "<u4").tobytes(), state=state.tobytes()).items()}
        self.scale = DK ** -0.5

    def buffers(self, tokens, seqs):
        rng, dt = self.rng, self.dt
        x = unpack_f32(pack_f32(rng.standard_normal((tokens, H)).astype(np.float32), dt), dt).reshape(tokens, H)
        g = -(0.05 * (0.2 + rng.random((tokens, HV)))).astype(np.float32)
        beta = (1 / (1 + np.exp(-rng.standard_normal((tokens, HV))))).astype(np.float32)
        given = rng.integers(0, VOCAB, (seqs, 1))
        self.host = dict(x=x, g=g, beta=beta, given=given)
        packed = dict(x=pack_f32(x, dt), g=g.tobytes(), beta=beta.tobytes(), given=given.astype("<u4").tobytes())
        if "rows" in self.b and self.b["rows"].nbytes == tokens * WIDTH * self.e:
            for k, v in packed.items():
                self.b[k].upload(v)
        else:
            sizes = dict(rows=tokens * WIDTH * self.e, y=tokens * HV * DV * 4, hidden=seqs * H * self.e, logits=seqs * VOCAB * self.e, lp=seqs * 4, ent=seqs * 4, ids=seqs * TOP * 4, top=seqs * TOP * 4)
            self.b.update({k: GpuBuffer.from_bytes(v) for k, v in packed.items()}, **{k: GpuBuffer(v) for k, v in sizes.items()})

    def run(self, lens, offsets):
        b, e, dt, n = self.b, self.e, self.dt, sum(lens)
        ops.fp8_qmv(dt, b["w_in"], b["s_in"], b["x"], b["rows"], n, WIDTH, H)
        at = b["rows"].ptr
        ops.gated_delta_rule(dt, at, at + HK * DK * e, at + 2 * HK * DK * e, b["g"], b["beta"], b["state"], b["state"], b["y"], len(lens), n, HK, HV, DK, DV, row_stride=WIDTH, offsets=offsets,
                             slots=b["slots"], n_slots=SLOTS, scale=self.scale, norm_eps=EPS)
        for i, last in enumerate(np.cumsum(lens) - 1):
            ops.gated_rms_norm_qmv(dt, 64, b["y"].ptr + int(last) * HV * DV * 4, at + (int(last) * WIDTH + WIDTH - HV * DV) * e, b["nw"], b["eps"], b["w4"], b["s4"], b["b4"], b["hidden"].ptr + i * H * e,
                                   HV, DV, H)
        ops.fp8_qmv(dt, b["w_head"], b["s_head"], b["hidden"], b["logits"], len(lens), VOCAB, H)
        ops.token_logprobs(dt, b["logits"], VOCAB, b["given"], 1, b["lp"], b["ent"], b["ids"], b["top"], TOP, len(lens), VOCAB)

    OUTPUTS = ("rows", "y", "state", "hidden", "logits", "lp", "ent", "ids", "top")

    def outputs(self):
        return {k: self.b[k].read_bytes() for k in self.OUTPUTS}

    def hold(self, lens, before):
        o, dt, n, seqs = self.outputs(), self.dt, sum(lens), len(lens)
        typed = lambda k, *shape: unpack_f32(o[k], dt).reshape(shape)
        f32 = lambda k, *shape: np.frombuffer(o[k], "<f4").reshape(shape)
        def product(x, w, s, got):
            xv, wv = ref.values(*ref.quantize(x, 1), 1), ref.values(w, s, 128)
            want = xv @ wv.T
            assert np.all(np.abs(got - want) <= _tolerance(xv, wv, want, dt, H))
        rows = typed("rows", n, WIDTH)
        product(self.host["x"], self.w_in, self.s_in, rows)
        q, k, v, z = (x.reshape(n, h, -1) for x, h in zip(np.split(rows, [HK * DK, 2 * HK * DK, 2 * HK * DK + HV * DV], 1), (HK, HK, HV, HV)))
        ends = np.cumsum(lens)
        wy, wS = rule(*(x.astype(np.float64) for x in (q, k, v, self.host["g"], self.host["beta"], before)), list(zip(ends - lens, ends)), self.slots, self.scale, EPS)
        rel = (DK / 16 + 16) * 2.0 ** -24 * max(lens)
        y = f32("y", n, HV, DV)
        assert np.all(np.abs(y - wy) <= rel * np.abs(wy).max()) and np.all(np.abs(f32("state", *before.shape) - wS) <= rel * np.abs(wS).max())
        untouched = [i for i in range(SLOTS) if i not in self.slots]
        assert np.array_equal(f32("state", *before.shape)[untouched], before[untouched])
        hidden = typed("hidden", seqs, H)
        for i, last in enumerate(ends - 1):
            _, want, _ = self.oracle.gated_rms_norm_qgemv(self.c.w, self.c.scales_f, self.c.biases_f, y[last].copy(), z[last].reshape(-1).copy(), self.nw, HV, DV, 64, H, np.float32(EPS))
            assert rel_err(hidden[i], self.oracle.round_through(want.astype(np.float32), ODT[dt])) <= TOL[dt]
        logits = typed("logits", seqs, VOCAB)
        product(hidden, self.w_head, self.s_head, logits)
        wlp, went, wids, wtop, size, d, zs = _reference(logits.astype(np.float64), self.host["given"], TOP)
        tol = lambda d: 1e-5 + 2.0 ** -22 * np.maximum(np.abs(d), np.log(VOCAB))
        assert _close(f32("lp", seqs, 1), wlp, tol(wlp)) and _close(f32("ent", seqs), went, 1e-5 * size) and _close(f32("top", seqs, TOP), wtop, tol(wtop))
        assert np.array_equal(np.frombuffer(o["ids"], "<u4").reshape(seqs, TOP), wids)

    def states(self):
        return np.frombuffer(self.b["state"].read_bytes(), "<f4").reshape(SLOTS, HV, DV, DK).copy()


@pytest.mark.parametrize("dt", [DType.F32, DType.F16, DType.BF16], ids=lambda d: d.name)
def test_prompt_and_tokens(oracle, dt):
    print(f"[case] linear attention step {dt.name}", flush=True)
    layer = Layer(oracle, dt)
    lens = [70, 1, 33]
    offsets = GpuBuffer.from_bytes(np.concatenate([[0], np.cumsum(lens)]).astype("<u4").tobytes())
    layer.buffers(sum(lens), 3)
    before = layer.states()
    layer.run(lens, offsets)
    layer.hold(lens, before)
    g, one = None, [1, 1, 1]
    try:
        for turn in range(4):
            layer.buffers(3, 3)
            before = layer.states()
            if g is None:
                layer.run(one, None)
                layer.hold(one, before)
                g = Graph()
                with g:
                    layer.run(one, None)
                continue
            g.replay()
            layer.hold(one, before)
            replayed = layer.outputs()
            layer.b["state"].upload(before.tobytes())
            layer.run(one, None)
            assert layer.outputs() == replayed
    finally:
        if g is not None:
            g.close()
