"""What the roundings of the attention over the 4-bit cache add up to, row by row and head by head: the length of the error's vector, not a worst case for each number.

Roundings to nearest are taken as independent, each of mean zero and at most u / sqrt(3) in the mean square of its value, u half a step of its type. With
p the weights, v the values and o the result:
  codes as operands   p s has u' (bf16 2^-8, f16 2^-16 in two terms): sum_j u'^2 p_j^2 |s (c - 8)_j|^2; and the result's u^2 |o|^2; all over 3
  keys, values and weights in T (prompts, f16 and bf16)
                      a key's roundings move a score by scale^2 sum_d q^2 k^2 u^2 in the mean square, and a score p (v - o): sum_j p_j^2 scale^2 sum_d (q k_j)^2 u^2 |v_j - o|^2;
                      a weight's and a value's: 2 sum_j p_j^2 u^2 |v_j|^2; the result's u^2 |o|^2; all over 3
A row is held to five times the root of that: sums of so many bounded terms pass five times theirs in less than one of a million. A whole call of many rows is held to the root itself,
which mantissas that are spread over their range leave 26 % below (0.74: the root of (1 - 1 / 4) / (2 ln 2)). What is f32 on the way, of 2^-24 each, comes on top in the same manner: a score
has dim / 8 + 24 roundings of at most |scale| |q| |k| (with codes as operands of 48 steps more for each of its dim terms); sums over n tokens n / 8 + 128 of at most p |v| (with
codes of 64 steps more). All in one direction: 2^-20 for the exponential.
"""
import numpy as np

from metaltile_amd import DType
from tests.kv_reference import HALF_STEP

HELD = {DType.F32: 2.0 ** -23, DType.F16: 2.0 ** -16, DType.BF16: 2.0 ** -8}


def attention(pool, q, offsets, hq, scale, window, dt, in_t):
    """(out [rows, hq, dim], bounds [rows, hq], bound of all) in 64 bits. Sequences hold at least as many tokens as rows, all on pages."""
    shared, u = hq // pool.hkv, HALF_STEP[dt]
    out, energy, sure = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for i, n in enumerate(pool.lens):
        rows = slice(offsets[i], offsets[i + 1])
        m = offsets[i + 1] - offsets[i]
        there, ((_, k), (vc, v)) = pool.of(i, n)
        assert m <= n <= pool.max_len and there.all()
        place, at = n - m + np.arange(m)[:, None], np.arange(n)[None]
        seen = (at <= place) & (at > place - window if window else True)
        for h in range(hq):
            x, kk, vv, cc = q[rows, h].astype(np.float64), k[h // shared], v[h // shared], vc[h // shared]
            s = np.where(seen, scale * (x @ kk.T), -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            p = e / e.sum(1, keepdims=True)
            o = p @ vv
            v2 = (vv * vv).sum(1)
            o2 = (o * o).sum(1)
            apart = v2[None] - 2 * (o @ vv.T) + o2[:, None]
            steps_k, steps_v = ((0 if in_t else 1) * _steps(pool, part, i, h // shared, n) for part in (0, 1))
            size = scale * scale * (x * x).sum(1)[:, None] * (48 * np.sqrt(pool.dim) * steps_k[:, 0] + np.linalg.norm(kk, axis=1)) ** 2
            sums = p @ (64 * steps_v + np.abs(vv))
            energy[rows, h] += 2.0 ** -48 * ((pool.dim / 8 + 24) * (p * p * size * apart).sum(1) + (seen.sum(1) / 8 + 128) * (sums * sums).sum(1))
            if in_t:
                energy[rows, h] += u * u * (p * p * (scale * scale * ((x * x) @ (kk * kk).T) * apart + 2 * v2)).sum(1)
            else:
                energy[rows, h] += HELD[dt] ** 2 * ((p * p) @ (cc * cc).sum(1))
            energy[rows, h] = (energy[rows, h] + u * u * o2) / 3
            sure[rows, h] = 2.0 ** -20 * (np.linalg.norm(p @ np.abs(vv), axis=1) + np.sqrt(o2))
            out[rows, h] = o
    return out, 5 * np.sqrt(energy) + sure, np.sqrt(energy.sum()) + np.sqrt((sure * sure).sum())


def _steps(pool, part, seq, head, n):
    at = np.arange(n)
    return np.abs(pool.parts[part][1][pool.pages[seq, at // pool.page], head, at % pool.page].astype(np.float64)).max(-1, keepdims=True)
