"""What the paged cache's calls and the norm would launch, and what they refuse: decided by shapes, so without a device. And what the Python calls hand over."""
import numpy as np
import pytest

from metaltile_amd import DType, ops

OK, BAD_ARG, SHAPE, UNSUPPORTED = 0, -2, -3, -7
DTYPES = [DType.F32, DType.F16, DType.BF16]
KV_OPS = ["kv_append", "kv_read", "kv_attention"]


def kv(op, dt=DType.BF16, max_len=100, group=64, hq=8, hkv=2, dim=128, seqs=3, tokens=6):
    return ops.plan(op, dt, max_len, group, hq, hkv, dim, seqs, tokens)


def _fits(rc, launches):
    assert rc in (OK, SHAPE) and (rc == OK) == bool(launches)
    for name, grid, block, lds in launches:
        assert name and all(0 < g * b < 1 << 32 for g, b in zip(grid, block)) and grid[1] <= 65535 and grid[2] == 1 and lds <= 160 * 1024
        assert block[0] * block[1] * block[2] <= 1024 and block[0] % 64 == 0


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("op", KV_OPS)
def test_launches(dt, op):
    rng = np.random.default_rng(1)
    for _ in range(400):
        dim = int(rng.choice([64, 128, 256]))
        hkv = int(rng.integers(1, 17))
        rc, launches, scratch, count = kv(op, dt, int(2 ** rng.uniform(0, 21)), int(rng.choice([g for g in (32, 64, 128) if g <= dim])), hkv * int(rng.integers(1, 9)), hkv, dim,
                                          int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 18)))
        assert count == len(launches) and (op == "kv_attention" or scratch == 0)
        _fits(rc, launches)
        assert rc == OK


@pytest.mark.parametrize("op", KV_OPS)
def test_sizes_next_to_what_a_launch_can_have(op):
    rng = np.random.default_rng(2)
    for _ in range(400):
        hkv = int(2 ** rng.uniform(0, 16))
        rc, launches, _, _ = kv(op, hq=hkv * int(rng.integers(1, 3)) if hkv < 30000 else hkv, hkv=hkv, tokens=min((1 << 24) - 1, int(2 ** rng.uniform(10, 24))), seqs=int(2 ** rng.uniform(0, 20)),
                                max_len=int(2 ** rng.uniform(0, 30)))
        _fits(rc, launches)


@pytest.mark.parametrize("op", KV_OPS)
def test_refusals(op):
    assert kv(op)[0] == OK
    assert kv(op, dt=5)[0] == BAD_ARG
    assert kv(op, dim=96, group=32)[0] == UNSUPPORTED and kv(op, dim=0)[0] == UNSUPPORTED
    assert kv(op, group=16)[0] == SHAPE and kv(op, group=0)[0] == SHAPE and kv(op, dim=64, group=128)[0] == SHAPE
    assert kv(op, hkv=0)[0] == SHAPE and kv(op, hkv=65537)[0] == SHAPE
    assert kv(op, tokens=1 << 24)[0] == SHAPE and kv(op, seqs=1 << 24)[0] == SHAPE
    assert kv(op, max_len=(1 << 30) + 16)[0] == SHAPE
    assert kv(op, tokens=0) == (OK, [], 0, 0) and kv(op, seqs=0, tokens=0) == (OK, [], 0, 0)
    if op == "kv_attention":
        assert kv(op, hq=0)[0] == SHAPE and kv(op, hq=3)[0] == SHAPE and kv(op, hq=65538)[0] == SHAPE


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_norm(dt):
    rng = np.random.default_rng(3)
    plan = lambda rows, cols, d=dt: ops.plan("add_rms_norm_fp8", d, 0, 0, rows, 0, cols)
    for _ in range(300):
        rc, launches, scratch, count = plan(int(2 ** rng.uniform(0, 28)), 16 * int(2 ** rng.uniform(0, 26)))
        _fits(rc, launches)
        assert scratch == 0 and count == len(launches)
    assert plan(0, 128) == (OK, [], 0, 0)
    assert plan(4, 0)[0] == SHAPE and plan(4, 24)[0] == SHAPE and plan(1 << 28, 16)[0] == SHAPE and plan(1 << 27, 128 * 16)[0] == SHAPE and plan(4, 0xFFFFFFF0)[0] == SHAPE
    assert plan(4, 128, 9)[0] == BAD_ARG


class _Library:
    def __getattr__(self, name):
        def call(*args):
            self.called, self.args = name, args
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(ops, "_ensure_init", lambda: lib)
    return lib


def test_what_is_handed_over(library):
    cache = ops.KvCache(1, 2, 3, 4, 5, 6, 10, 16, 2, 128, 64)
    batch = ops.KvBatch(7, 9, 8, 3, 6, 100)
    assert (cache.k_codes, cache.v_biases, cache.n_pages, cache.page_size, cache.n_heads, cache.head_dim, cache.group_size) == (1, 6, 10, 16, 2, 128, 64)
    assert (batch.pages, batch.offsets, batch.lens, batch.pages_stride, batch.n_seqs, batch.n_tokens, batch.max_len) == (7, None, 8, 9, 3, 6, 100)
    assert ops.KvBatch(7, 9, 8, 3, 6, 100, offsets=11).offsets == 11
    for stride, want in ((None, (1024, 256, 256)), (2000, (2000,) * 3), (np.int64(2000), (2000,) * 3), ([1, 2, 3], (1, 2, 3)), (np.array([1, 2, 3]), (1, 2, 3))):
        ops.kv_append(DType.BF16, cache, batch, 20, 21, row_stride=stride, q=22, q_out=23, hq=8, cos_sin=24, n_positions=100, rot=64, neighbours=True)
        assert library.called == "mtq_kv_append" and library.args[3:] == (22, want[0], 23, 1024, 8, 20, want[1], 21, want[2], 24, 100, 64, 1)
    ops.kv_append(DType.BF16, cache, batch, 20, 21)
    assert library.args[3:] == (None, 0, None, 0, 0, 20, 256, 21, 256, None, 0, 0, 0)
    ops.kv_read(DType.F16, cache, batch, None, 5)
    assert library.args[3:] == (None, 5)
    ops.kv_attention(DType.F16, cache, batch, 30, 31, 8, 0.5, window=4)
    assert library.args[3:] == (30, 1024, 31, 1024, 8, 0.5, 4)
    ops.kv_attention(DType.F16, cache, batch, 30, 31, 8, 0.5, q_stride=1536, out_stride=1040)
    assert library.args[3:] == (30, 1536, 31, 1040, 8, 0.5, 0)
    ops.add_rms_norm_fp8(DType.F32, 1, None, 2, 1e-5, None, 3, 4, 5, 128)
    assert library.args == (0, 1, None, 2, 1e-5, None, 3, 4, 5, 128)
