"""The gated delta rule against 64 bits.

Tolerance. A token's products with the state have dk terms in f32 sums of dk / 16 in a row and four additions across lanes (or blocks of as
many on the matrix cores): relative to the magnitudes that enter, (dk / 16 + 4) 2^-24; decay, update and norms add less than 12 roundings. With q, k of
norm one or less and beta in (0, 1) a token's step makes no error before it larger, and the decay exp(g) shrinks it, so that errors of at most
min(tokens, 1 / (1 - max exp(g))) tokens add up: (dk / 16 + 16) 2^-24 x that many x the largest value of the reference.
"""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests.hip_graph import Graph

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]
EPS = 1e-6


def rule(q, k, v, g, beta, S, bounds, slots, scale, eps):
    """y [tokens, hv, dv] and states, f64; bounds: [(from, to)]."""
    hv, hk = v.shape[1], q.shape[1]
    q, k = (np.repeat(x, hv // hk, 1) for x in (q, k))
    if eps >= 0:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    y, S = np.zeros(v.shape), S.copy()
    for (lo, hi), slot in zip(bounds, slots):
        if slot >= S.shape[0]:
            continue
        s = S[slot]
        for t in range(lo, hi):
            s = s * np.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - np.einsum("hvk,hk->hv", s, k[t]))
            s = s + u[:, :, None] * k[t][:, None, :]
            y[t] = scale * np.einsum("hvk,hk->hv", s, q[t])
        S[slot] = s
    return y, S


class Case:
    def __init__(self, dt, lens, hk, hv, dk, dv, seed=0, eps=EPS, decay=0.05, slots=None, n_slots=None, apart=False, tail=0, equal=False, fresh=False):
        rng = np.random.default_rng(seed + sum(lens) + dk)
        self.dt, self.lens, self.hk, self.hv, self.dk, self.dv, self.eps, self.equal, self.fresh = dt, lens, hk, hv, dk, dv, eps, equal, fresh
        self.tokens = sum(lens) + tail
        self.scale = dk ** -0.5
        typed = lambda x: unpack_f32(pack_f32(x.astype(np.float32), dt), dt).reshape(x.shape)
        n = self.tokens
        self.q, self.k, self.v = (typed(rng.standard_normal((n, h, d)) * s) for h, d, s in ((hk, dk, 1), (hk, dk, 1 if eps >= 0 else dk ** -0.5), (hv, dv, 1)))
        self.g = -(decay * (0.2 + rng.random((n, hv)))).astype(np.float32)
        self.beta = (1 / (1 + np.exp(-rng.standard_normal((n, hv))))).astype(np.float32)
        self.n_slots = n_slots or len(lens)
        self.slots = slots
        self.state = (0.3 * rng.standard_normal((self.n_slots, hv, dv, dk))).astype(np.float32)
        self.offsets = np.concatenate([[0], np.cumsum(lens)]).astype("<u4")
        if apart:   # three buffers, rows of odd lengths
            self.strides = (hk * dk + 3, hk * dk + 1, hv * dv + 5)
            parts = [np.full((n, s), np.nan, np.float32) for s in self.strides]
            for p, x in zip(parts, (self.q, self.k, self.v)):
                p[:, :x[0].size] = x.reshape(n, -1)
            self.bufs = [GpuBuffer.from_bytes(pack_f32(p, dt)) for p in parts]
            self.at = [b.ptr for b in self.bufs]
        else:       # side by side in one row
            w = 2 * hk * dk + hv * dv
            self.strides = (w, w, w)
            rows = np.concatenate([x.reshape(n, x.shape[1] * x.shape[2]) for x in (self.q, self.k, self.v)], 1)
            self.bufs = [GpuBuffer.from_bytes(pack_f32(rows, dt) or bytes(4))]
            e = dt.size_bytes
            self.at = [self.bufs[0].ptr, self.bufs[0].ptr + hk * dk * e, self.bufs[0].ptr + 2 * hk * dk * e]
        self.gb, self.bb, self.ob = (GpuBuffer.from_bytes(x.tobytes() or bytes(4)) for x in (self.g, self.beta, self.offsets))
        self.sb = None if slots is None else GpuBuffer.from_bytes(np.array(slots, "<u4").tobytes())
        self.state_in = GpuBuffer.from_bytes(self.state.tobytes())
        self.state_out = GpuBuffer.from_bytes(np.full(self.state.size, 7.5, "<f4").tobytes())
        self.y = GpuBuffer.from_bytes(np.full(max(1, n * hv * dv), 9.5, "<f4").tobytes())

    def call(self, in_place=False):
        ops.gated_delta_rule(self.dt, *self.at, self.gb, self.bb, None if self.fresh else self.state_in, self.state_in if in_place else self.state_out, self.y, len(self.lens), self.tokens,
                             self.hk, self.hv, self.dk, self.dv, row_stride=self.strides, offsets=None if self.equal else self.ob, slots=self.sb, n_slots=self.n_slots,
                             scale=self.scale, norm_eps=self.eps)

    def results(self, in_place=False):
        y = np.frombuffer(self.y.read_bytes(), "<f4")[:self.tokens * self.hv * self.dv].reshape(self.tokens, self.hv, self.dv)
        return y, np.frombuffer((self.state_in if in_place else self.state_out).read_bytes(), "<f4").reshape(self.state.shape)

    def hold(self, in_place=False):
        y, S = self.results(in_place)
        bounds = list(zip(self.offsets[:-1], self.offsets[1:]))
        slots = self.slots or range(len(self.lens))
        start = np.zeros(self.state.shape) if self.fresh else self.state.astype(np.float64)
        wy, wS = rule(*(x.astype(np.float64) for x in (self.q, self.k, self.v, self.g, self.beta)), start, bounds, slots, self.scale, self.eps)
        done = np.zeros(self.tokens, bool)
        named = np.zeros(self.n_slots, bool)
        for (lo, hi), slot in zip(bounds, slots):
            if slot < self.n_slots:
                done[lo:hi] = named[slot] = True
        reach = min(max(self.lens, default=0), 1 / (1 - np.exp(self.g.max())) if self.g.size else 1) if self.g.size and self.g.max() < 0 else max(self.lens, default=0)
        rel = (self.dk / 16 + 16) * 2.0 ** -24 * max(reach, 1)
        if done.any():
            assert np.all(np.abs(y[done] - wy[done]) <= rel * np.abs(wy[done]).max() + 1e-30), float(np.abs(y[done] - wy[done]).max() / np.abs(wy[done]).max())
        assert np.all(y[~done] == 9.5)
        if named.any():
            assert np.all(np.abs(S[named] - wS[named]) <= rel * max(np.abs(wS[named]).max(), 1e-30)), float(np.abs(S[named] - wS[named]).max() / np.abs(wS[named]).max())
        assert np.all(S[~named] == (self.state[~named] if in_place else 7.5))


SHAPES = [  # lens, hk, hv, dk, dv
    ([1], 1, 1, 128, 128), ([1], 16, 32, 128, 128), ([1] * 5, 2, 6, 64, 128), ([2], 1, 1, 1, 1), ([3], 2, 2, 7, 5), ([4, 1], 1, 3, 100, 36), ([5], 2, 4, 256, 64), ([1, 6], 1, 2, 200, 130),
    ([0, 3, 0, 1], 2, 2, 64, 64), ([63], 1, 2, 128, 128), ([64], 1, 2, 128, 128), ([65], 2, 2, 128, 64), ([128, 1, 0, 130], 1, 2, 64, 128), ([200], 1, 1, 64, 64), ([129], 1, 2, 128, 16),
    ([17, 300], 2, 4, 128, 128), ([70, 90], 1, 1, 96, 48), ([100], 1, 1, 256, 256), ([500], 1, 3, 128, 128), ([257], 2, 4, 128, 80), ([191, 64, 2], 1, 1, 32, 32)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,hk,hv,dk,dv", SHAPES, ids=lambda v: str(v).replace(" ", ""))
def test_against_64_bits(dt, lens, hk, hv, dk, dv):
    print(f"[case] gated_delta_rule {dt.name} lens{lens} hk{hk} hv{hv} dk{dk} dv{dv}", flush=True)
    c = Case(dt, lens, hk, hv, dk, dv)
    c.call()
    c.hold()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens", [[1, 1, 1], [2, 90, 0, 70]], ids=str)
@pytest.mark.parametrize("how", ["apart", "slots", "missing_slot", "in_place", "fresh", "raw", "tail", "strong_decay", "no_decay"])
def test_ways_to_call(dt, lens, how):
    print(f"[case] gated_delta_rule {dt.name} lens{lens} {how}", flush=True)
    n = len(lens)
    kw = {"apart": dict(apart=True), "slots": dict(slots=[(2 * i + 1) % (n + 3) for i in range(n)], n_slots=n + 3), "missing_slot": dict(slots=[0xFFFFFFFF if i == 1 else i for i in range(n)]),
          "in_place": {}, "fresh": dict(fresh=True), "raw": dict(eps=-1.0), "tail": dict(tail=67), "strong_decay": dict(decay=40.0), "no_decay": dict(decay=0.0)}[how]
    c = Case(dt, lens, 2, 4, 128, 64, **kw)
    c.call(how == "in_place")
    c.hold(how == "in_place")


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [80, 80], [0, 0]], ids=str)
def test_equal_lengths_without_offsets(lens):
    c = Case(DType.BF16, lens, 1, 2, 128, 128, equal=True)
    c.call()
    c.hold()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_repeated_and_extreme_rows(dt):
    """Keys that are all the same (beta 1: each value replaces the last), zero rows (over a norm of sqrt(eps)), magnitudes far from one."""
    c = Case(dt, [150], 1, 2, 128, 64, seed=3)
    for kind in ("same", "zero", "large", "small"):
        k, v, beta = c.k.copy(), c.v.copy(), c.beta.copy()
        if kind == "same": k[:] = k[0]; beta[:] = 1
        elif kind == "zero": k[::3] = 0; c.q[::5] = 0
        elif kind == "large": k *= 64; v *= 1024
        else: k /= 64; v /= 1024
        typed = lambda x: unpack_f32(pack_f32(x.astype(np.float32), dt), dt).reshape(x.shape)
        c.k, c.v, c.beta = typed(k), typed(v), beta.astype(np.float32)
        rows = np.concatenate([x.reshape(c.tokens, -1) for x in (c.q, c.k, c.v)], 1)
        c.bufs[0].upload(pack_f32(rows, dt))
        c.bb.upload(c.beta.tobytes())
        c.call()
        c.hold()


@pytest.mark.parametrize("cut", [1, 64, 100, 299])
def test_a_sequence_in_two_calls(cut):
    """The state of the first call is where the second goes on."""
    whole = Case(DType.BF16, [300], 1, 2, 128, 128, seed=5)
    whole.call()
    y, S = whole.results()
    c, n = whole, 300
    e, w = 2, c.strides[0]
    state, out = GpuBuffer.from_bytes(c.state.tobytes()), GpuBuffer(4 * n * c.hv * c.dv)
    for lo, hi in ((0, cut), (cut, n)):
        ops.gated_delta_rule(c.dt, *(a + lo * w * e for a in c.at), c.gb.ptr + 4 * lo * c.hv, c.bb.ptr + 4 * lo * c.hv, state, state, out.ptr + 4 * lo * c.hv * c.dv, 1, hi - lo, c.hk, c.hv,
                             c.dk, c.dv, row_stride=w, scale=c.scale, norm_eps=EPS)
    y2 = np.frombuffer(out.read_bytes(), "<f4").reshape(y.shape)
    S2 = np.frombuffer(state.read_bytes(), "<f4").reshape(S.shape)
    rel = 2 * (8 + 16) * 2.0 ** -24 / (1 - np.exp(c.g.max()))
    assert np.abs(y - y2).max() <= rel * np.abs(y).max() and np.abs(S - S2).max() <= rel * np.abs(S).max()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("most_kb", [1, 200, 400, 1000])
def test_little_scratch(dt, most_kb):
    """Chunks in windows of as many as fit the scratch that the caller allows, token by token where none does."""
    lib = _ensure_init()
    _lib.check(lib.mtq_set_option(b"scratch.most_kb", most_kb))
    try:
        for lens in ([300], [70, 5, 0, 130, 64], [3, 200, 0]):
            c = Case(dt, lens, 1, 2, 64, 48)
            c.call()
            c.hold()
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))


def test_refusals():
    c = Case(DType.BF16, [4, 4], 2, 4, 64, 64)
    ok = dict(n_seqs=2, n_tokens=8, hk=2, hv=4, dk=64, dv=64, row_stride=512, offsets=c.ob, n_slots=2, q=c.at[0], k=c.at[1], v=c.at[2], g=c.gb, beta=c.bb, out=c.state_out, y=c.y, dt=DType.BF16)
    for bad in (dict(hk=3), dict(hk=0), dict(hv=0), dict(dk=0), dict(dk=257), dict(dv=0), dict(row_stride=127), dict(row_stride=(128, 128, 255)), dict(n_slots=1), dict(offsets=None, n_tokens=7), dict(q=0),
                dict(k=0), dict(v=0), dict(g=0), dict(beta=0), dict(out=0), dict(y=0), dict(dt=4)):
        a = dict(ok, **bad)
        with pytest.raises(MtqError):
            ops.gated_delta_rule(a["dt"], a["q"], a["k"], a["v"], a["g"], a["beta"], None, a["out"], a["y"], a["n_seqs"], a["n_tokens"], a["hk"], a["hv"], a["dk"], a["dv"], row_stride=a["row_stride"],
                                 offsets=a["offsets"], n_slots=a["n_slots"])


def test_offsets_behind_the_tokens():
    """Offsets past n_tokens, or that fall: no token outside is read or written."""
    c = Case(DType.BF16, [10, 20], 1, 2, 64, 64, tail=0)
    c.ob.upload(np.array([0, 10, 4000], "<u4").tobytes())
    c.call()
    c.hold()
    c.ob.upload(np.array([40, 35, 30], "<u4").tobytes())
    c.y.upload(np.full(c.tokens * c.hv * c.dv, 9.5, "<f4").tobytes())
    c.call()
    y, S = c.results()
    assert np.all(y == 9.5) and np.array_equal(S, c.state)


@pytest.mark.parametrize("lens", [[1, 1], [100, 40]], ids=str)
def test_captured(lens):
    c = Case(DType.BF16, lens, 1, 2, 128, 128)
    g = Graph()
    try:
        with g:
            c.call()
        for turn in range(3):
            c.state = (0.3 * np.random.default_rng(turn).standard_normal(c.state.shape)).astype(np.float32)
            c.state_in.upload(c.state.tobytes())
            g.replay()
            c.hold()
            first = [x.copy() for x in c.results()]
            c.call()
            assert all(np.array_equal(a, b) for a, b in zip(first, c.results()))
    finally:
        g.close()
