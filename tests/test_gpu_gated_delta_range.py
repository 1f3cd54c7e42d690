"""The gated delta rule where f32 ends inside a chunk, from inputs that are all finite: tokens before that place are what they are without it, and
the result does not depend on whether a sequence goes in chunks or token by token.

Tolerances are those of test_gpu_gated_delta.py: (dk / 16 + 16) 2^-24 x the tokens whose errors add up x the largest value of the reference. Where the
recurrence grows, a token's error is carried on and grows with the values, so that it stays in proportion to the largest value so far.
"""
import numpy as np
import pytest

from metaltile_amd import DType, _lib, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests.test_gpu_gated_delta import Case, rule

pytestmark = pytest.mark.gpu
DTYPES = [DType.F32, DType.F16, DType.BF16]


def _put(c):
    """The case's inputs as they are now, rounded to its type."""
    typed = lambda x: unpack_f32(pack_f32(x.astype(np.float32), c.dt), c.dt).reshape(x.shape)
    c.q, c.k, c.v = typed(c.q), typed(c.k), typed(c.v)
    c.bufs[0].upload(pack_f32(np.concatenate([x.reshape(c.tokens, -1) for x in (c.q, c.k, c.v)], 1), c.dt))
    c.gb.upload(c.g.tobytes())
    c.bb.upload(c.beta.tobytes())


def _both_ways(c):
    """Results in chunks, and token by token (no scratch for chunks)."""
    lib, out = _ensure_init(), []
    for most_kb in (0, 1):
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", most_kb))
        try:
            c.call()
        finally:
            _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))
        out.append([x.copy() for x in c.results()])
    return out


@pytest.mark.parametrize("dt", [DType.F32, DType.BF16], ids=lambda d: d.name)
@pytest.mark.parametrize("what", ["k", "q", "both"])
def test_squares_past_the_range(dt, what):
    """Keys and queries of 3e19, whose squares are infinite: they count as zeros, and every other token is what it is with zeros in their place."""
    c = Case(dt, [150, 40], 1, 2, 128, 64, seed=11)
    at = [70, 75, 90, 130, 160, 165]
    for x in {"k": (c.k,), "q": (c.q,), "both": (c.q, c.k)}[what]:
        x[at] = 3e19 * np.sign(x[at])
    _put(c)
    chunks, tokens = _both_ways(c)
    for x in (c.q, c.k):
        x[np.abs(x).max(-1) > 1e19] = 0
    wy, wS = rule(*(x.astype(np.float64) for x in (c.q, c.k, c.v, c.g, c.beta, c.state)), list(zip(c.offsets[:-1], c.offsets[1:])), range(2), c.scale, c.eps)
    rel = (128 / 16 + 16) * 2.0 ** -24 * min(150, 1 / (1 - np.exp(c.g.max())))
    for y, S in (tokens, chunks):
        assert np.all(np.abs(y - wy) <= rel * np.abs(wy).max()) and np.all(np.abs(S - wS) <= rel * np.abs(wS).max())


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,begin", [([60], 30), ([200, 64], 97), ([64], 1), ([130], 129)], ids=str)
def test_a_recurrence_that_leaves_the_range(dt, lens, begin):
    """Keys as they are; from token `begin` on one key whose squares sum up to 128, so that each token makes the state 63 times larger until f32 ends,
    some twenty tokens later. The other sequence is what it is alone."""
    n = lens[0]
    c = Case(dt, lens, 1, 2, 128, 64, seed=13, eps=-1.0)
    c.k[begin:n] = np.where(c.k[begin] < 0, -1, 1)
    c.beta[begin:n] = 0.5
    _put(c)
    chunks, tokens = _both_ways(c)
    wy, wS = rule(*(x.astype(np.float64) for x in (c.q, c.k, c.v, c.g, c.beta, c.state)), list(zip(c.offsets[:-1], c.offsets[1:])), range(len(lens)), c.scale, c.eps)
    # Sums of 128 products with such a key have magnitudes of sqrt(128) |S| and more where the sum itself is |S|: as many times the roundings.
    reach = 1 / (1 - np.exp(c.g.max()))
    rel = lambda tokens: 128 ** 0.5 * (128 / 16 + 16) * 2.0 ** -24 * tokens
    for y, S in (tokens, chunks):
        for t in range(min(n, begin + 15)):        # (63^15 is 1e27)
            assert np.all(np.abs(y[t] - wy[t]) <= rel(reach + 1 + max(0, t - begin)) * np.abs(wy[t if t >= begin else 0:t + 1]).max()), t
        assert n < begin + 25 or np.abs(wy[begin + 25:n]).max(-1).min() > 1e39 and not np.isfinite(y[begin + 25:n]).any()
        assert np.all(np.abs(y[n:] - wy[n:]) <= rel(reach) * np.abs(wy[n:]).max(initial=0))
        if len(lens) > 1:
            assert np.all(np.abs(S[1] - wS[1]) <= rel(reach) * np.abs(wS[1]).max())


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_decays_that_grow(dt):
    """A decay that lets the state grow by e^100 inside a chunk: the tokens before it keep their values."""
    c = Case(dt, [100], 1, 2, 64, 32, seed=17)
    c.g[20], c.g[40], c.g[50] = -100.0, 100.0, -100.0
    _put(c)
    wy, wS = rule(*(x.astype(np.float64) for x in (c.q, c.k, c.v, c.g, c.beta, c.state)), [(0, 100)], [0], c.scale, c.eps)
    rel = (64 / 16 + 16) * 2.0 ** -24 * 40
    for y, S in _both_ways(c):
        assert np.all(np.abs(y[:40] - wy[:40]) <= rel * np.abs(wy[:40]).max())
