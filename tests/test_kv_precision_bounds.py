"""What the bounds of kv_precision find: mistakes planted in the oracle's result, on the host."""
import numpy as np
import pytest

from metaltile_amd import DType
from tests import kv_precision
from tests import kv_reference as ref
from tests.kv_reference import typed

CASES = [  # lens, rows, window, dim, group, query heads, key heads
    ([300], [200], 17, 128, 64, 4, 2), ([300, 70], [200, 70], 64, 64, 64, 4, 2), ([300], [200], 64, 256, 32, 2, 1), ([200], [77], 0, 128, 128, 2, 2), ([200], [100], 0, 64, 32, 4, 1)]


@pytest.mark.parametrize("dt", [DType.F16, DType.BF16], ids=lambda d: d.name)
@pytest.mark.parametrize("in_t", [True, False])
@pytest.mark.parametrize("lens,rows,window,dim,group,hq,hkv", CASES, ids=str)
def test_planted_mistakes(dt, in_t, lens, rows, window, dim, group, hq, hkv):
    rng = np.random.default_rng(1)
    pool = ref.Pool(dt, rng, lens, hkv, dim, group, 16)
    offsets = np.concatenate([[0], np.cumsum(rows)]).tolist()
    q = typed(rng.standard_normal((offsets[-1], hq, dim)), dt)
    oracle = lambda w: kv_precision.attention(pool, q, offsets, hq, dim ** -0.5, w, dt, in_t)  # noqa: E731
    want, each, of_all = oracle(window)
    length = np.linalg.norm(want, axis=2)
    assert of_all < {DType.F16: 0.002, DType.BF16: 0.008}[dt] * np.linalg.norm(want)

    def found(got):
        """Of the rows that differ, how many pass their bound; and the whole difference against its bound."""
        far = np.linalg.norm(got - want, axis=2)
        return (far > each)[far > 0].mean(), np.linalg.norm(got - want) / of_all

    assert found(np.zeros_like(want))[0] == 1
    noise = rng.standard_normal(want.shape)
    rows_found, whole = found(want + 0.1 * noise * (length / np.linalg.norm(noise, axis=2))[..., None])
    assert rows_found == 1 and whole > 8
    # A token more and one fewer: of a window's, or of what the last rows see.
    if window:
        for w in (window - 1, window + 1):
            rows_found, whole = found(oracle(w)[0])
            assert rows_found > 0.4 and whole > 8
    else:
        rows_found, whole = found(oracle(max(lens) - 20)[0])   # (20 rows have lost their first tokens)
        assert rows_found > 0.7 and whole > 4


def test_roundings_as_they_are_pass():
    """Keys, values, weights and the result rounded on the host: within the bounds, and not far below the whole one."""
    for dt in (DType.F16, DType.BF16):
        rng = np.random.default_rng(3)
        pool = ref.Pool(dt, rng, [260], 1, 128, 64, 16)
        q = typed(rng.standard_normal((120, 2, 128)), dt)
        want, each, of_all = kv_precision.attention(pool, q, [0, 120], 2, 128 ** -0.5, 0, dt, True)
        _, ((_, k), (_, v)) = pool.of(0, 260)
        got = np.zeros_like(want)
        for h in range(2):
            s = q[:, h].astype(np.float64) @ typed(k[0], dt).astype(np.float64).T * 128 ** -0.5
            s = np.where(np.arange(260) <= np.arange(140, 260)[:, None], s, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True)) * 2.0 ** 11
            got[:, h] = typed((typed(e, dt).astype(np.float64) @ typed(v[0], dt)) / e.sum(1, keepdims=True), dt)
        assert np.all(np.linalg.norm(got - want, axis=2) <= each)
        assert 0.4 * of_all < np.linalg.norm(got - want) <= of_all
