"""The gated delta rule in chunks holds f32 accuracy: its operands are sums of three bf16 terms (f16: of their own two, bf16: one), and none may be lost.

Bound on the 2-norm of the error, for y and for the states, as a part of the result's. A value has about dk / 16 + 16 roundings behind it (sums of dk products
in blocks, decay, norms, updates), each 2^-24 of its size at most and 2^-24 / sqrt(3) in the mean square, independent: sqrt(dk / 16 + 16) of these. What the
tokens before left in the state stands to it as they do, and is not amplified (beta in (0, 1), keys of norm one). Four times that is allowed: 6.7e-7 for dk =
128. An operand of two terms keeps 16 bits and is off by up to 2^-17 = 7.6e-6 of its values, which test_bound shows to be past the bound in the result, for
every operand of the form in chunks.
"""
import numpy as np
import pytest

from metaltile_amd import DType
from tests.test_gpu_gated_delta import Case, rule

DTYPES = [DType.F32, DType.F16, DType.BF16]
CHUNK = 64


def bound(dk):
    return 4 * (dk / 16 + 16) ** 0.5 * 2.0 ** -24 / 3 ** 0.5


def _off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def _bf16(x):
    u = np.float32(x).view(np.uint32).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def _terms(x, n):
    total, rest = np.zeros_like(x, dtype=np.float32), np.array(x, np.float32)
    for _ in range(n):
        t = _bf16(rest)
        total, rest = total + t, rest - t
    return total


def _in_chunks(q, k, v, g, beta, S, scale, eps, cut):
    """One head in f32, chunk by chunk; the operand named `cut` has two bf16 terms, the others three."""
    f = np.float32
    held = lambda name, x: _terms(x, 2 if name == cut else 3)
    rk, rq = (f(s) / np.sqrt((x * x).sum(-1) + f(eps)) for s, x in ((1, k), (scale, q)))
    y = []
    for a in range(0, len(q), CHUNK):
        at = slice(a, a + CHUNK)
        K, Q, G, r, p, b = k[at], q[at], np.cumsum(g[at].astype(np.float64)), rk[at], rq[at], beta[at]
        D = np.tril(np.exp(G[:, None] - G[None, :])).astype(f)
        A = np.tril(b[:, None] * r[:, None] * r[None, :] * D * (K @ K.T), -1)
        P = p[:, None] * r[None, :] * D * (Q @ K.T)
        T = (np.linalg.inv(np.eye(len(K)) + A.astype(np.float64)) * b[None, :]).astype(f)
        e = np.exp(G).astype(f)
        X = v[at] - (e * r)[:, None] * (K @ held("S", S).T)
        U = held("T", T) @ held("X", X)
        y.append((e * p)[:, None] * (Q @ held("S", S).T) + held("P", P) @ held("U", U))
        W = (r * np.exp(G[-1] - G).astype(f))[:, None] * U
        S = e[-1] * S + (K.T @ held("W", W)).T
    return np.concatenate(y), S


@pytest.mark.parametrize("decay", [0.05, 0.0])
def test_bound(decay):
    """On the host: f32 is well inside the bound, and an operand of two terms outside."""
    rng = np.random.default_rng(5)
    n, dk, dv, eps, scale = 300, 128, 64, 1e-6, np.float32(128 ** -0.5)
    q, k = (_bf16(rng.standard_normal((n, dk))) for _ in range(2))
    v, S = _bf16(rng.standard_normal((n, dv))), (0.3 * rng.standard_normal((dv, dk))).astype(np.float32)
    g, beta = -(decay * (0.2 + rng.random(n))).astype(np.float32), (1 / (1 + np.exp(-rng.standard_normal(n)))).astype(np.float32)
    wide = [x.astype(np.float64) for x in (q[:, None], k[:, None], v[:, None], g[:, None], beta[:, None], S[None, None])]
    wy, wS = rule(*wide, [(0, n)], [0], float(scale), eps)
    for cut in (None, "S", "T", "X", "P", "U", "W"):
        y, last = _in_chunks(q, k, v, g, beta, S, scale, eps, cut)
        off = max(_off(y, wy[:, 0]), _off(last, wS[0, 0]))
        assert off < 0.6 * bound(dk) if cut is None else off > 1.5 * bound(dk), (cut, off)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("decay", [0.05, 0.0])
@pytest.mark.parametrize("lens,dk", [([63], 128), ([129], 128), ([100, 64, 300], 128), ([500], 64), ([1000], 128), ([200], 256)], ids=str)
def test_chunks(dt, decay, lens, dk):
    print(f"[case] gated_delta_rule {dt.name} lens{lens} dk{dk} decay{decay}", flush=True)
    c = Case(dt, lens, 2, 4, dk, 64, seed=21, decay=decay)
    c.call()
    y, S = c.results()
    wy, wS = rule(*(x.astype(np.float64) for x in (c.q, c.k, c.v, c.g, c.beta, c.state)), list(zip(c.offsets[:-1], c.offsets[1:])), range(len(lens)), c.scale, c.eps)
    off = [_off(y[lo:hi], wy[lo:hi]) for lo, hi in zip(c.offsets[:-1], c.offsets[1:])] + [_off(S[i], wS[i]) for i in range(len(lens))]
    print(f"off by {max(off):.2e}, bound {bound(dk):.2e}", flush=True)
    assert max(off) <= bound(dk)
