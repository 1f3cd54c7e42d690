"""Attention where one token has nearly all of the weight and a value of zero, so that the result is what thousands of others add up to (a first token that draws the attention
of all heads is such a one). Their weights, 2^-11.5 to 2^-24.5 of the largest, are held as finely as large ones.

Tolerance, relative: a weight's rounding and the result's (half a step of T each), a score's roundings twice (2 (64 + 24) 2^-24 of |scale| sum |q| (48 s + |k|) = 64 (48 s + |k|)), 2^-19
for the exponential, f32 sums over n tokens (n / 8 + 128) 2^-24 with values' codes (their scale's share of a value, 64 s), and half a step of p s times 8 s. In f16 a result below
2^-14 has steps of 2^-24.
"""
import numpy as np
import pytest

from metaltile_amd import DType, pack_f32
from tests.kv_reference import DTYPES, HALF_STEP
from tests.test_gpu_kv_attention import Attention, option  # noqa: F401

pytestmark = pytest.mark.gpu
TOKENS, ROWS, STEP = 12000, 100, 2.0 ** -10


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("top,rest", [(0.125, 0.0), (0.125, -0.0625), (0.125, -0.109375), (0.125, -0.140625)], ids=str)
@pytest.mark.parametrize("kernel,slices", [(0, 0), (1, 3), (2, 1), (4, 1), (4, 5)], ids=str)
def test_what_many_small_weights_add_up_to(dt, dim, top, rest, kernel, slices, option):  # noqa: F811
    print(f"[case] kv_attention small weights {dt.name} {dim} {rest} kernel {kernel} slices {slices}", flush=True)
    c = Attention(dt, [TOKENS], [ROWS], hq=2, hkv=1, dim=dim, scale=64 / dim)
    (kc, ks, kb), (vc, vs, vb) = c.pool.parts
    for codes, scales in ((kc, ks), (vc, vs)):
        codes[:], scales[:] = 0, STEP
    kb[:], vb[:] = rest, 1.0
    first = c.pool.pages[0, 0], slice(None), 0
    kb[first], vb[first], vs[first] = top, 0.0, 0.0
    for i, (codes, scales, biases) in enumerate(c.pool.parts):
        c.pool.bufs[3 * i].upload(np.zeros(c.pool.bufs[3 * i].nbytes, np.uint8))
        c.pool.bufs[3 * i + 1].upload(pack_f32(scales, dt))
        c.pool.bufs[3 * i + 2].upload(pack_f32(biases, dt))
    c.q[:] = 1.0
    c.upload()
    option("kv.kernel", kernel)
    option("kv.slices", slices)
    c.call()
    got = c.result().astype(np.float64)
    n = TOKENS - ROWS + np.arange(ROWS)   # tokens besides the first that a row sees
    mass = n * np.exp(64 * (rest - top))
    want = (mass / (1 + mass))[:, None, None]
    half = HALF_STEP[dt]
    rel = 2 * half + 2 * 88 * 2.0 ** -24 * 64 * (48 * STEP + abs(top)) + 2.0 ** -19 + (TOKENS / 8 + 128) * 2.0 ** -24 * (1 + 64 * STEP) + half * 8 * STEP
    tol = rel * want + (2.0 ** -25 if dt == DType.F16 else 0)
    far = np.abs(got - want) / tol
    assert np.all(far <= 1), f"{far.max()} of the tolerance"
