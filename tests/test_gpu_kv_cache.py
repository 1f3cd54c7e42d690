"""Writer and reader of the paged 4-bit cache: codes, scales and biases to the bit, what is not written, rotations of any width, order and stride."""
import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, ops, pack_f32, unpack_f32
from tests import kv_reference as ref
from tests.hip_graph import Graph
from tests.kv_reference import DTYPES, typed

pytestmark = pytest.mark.gpu


class Append:
    def __init__(self, dt, lens, rows, hq=4, hkv=2, dim=128, group=64, page=16, rot=None, neighbours=False, seed=1, pad=0, apart=False, gaps=False, max_len=None):
        self.dt, self.lens, self.hq, self.hkv, self.dim, self.group, self.neighbours = dt, lens, hq, hkv, dim, group, neighbours
        self.rot = rot = dim if rot is None else rot
        rng = self.rng = np.random.default_rng(seed)
        self.pool = ref.Pool(dt, rng, lens, hkv, dim, group, page, max_len=max_len)
        self.offsets = np.concatenate([[0], np.cumsum(rows)]).astype(int).tolist()
        if gaps:   # rows in front of the first sequence and behind the last
            self.offsets = [o + 3 for o in self.offsets]
        self.tokens = self.offsets[-1] + (2 if gaps else 0)
        n = self.tokens
        self.q, self.k, self.v = (typed(rng.standard_normal((n, h, dim)) * np.exp(rng.standard_normal((n, h, 1))), dt) for h in (hq, hkv, hkv))
        angle = np.arange(max(self.pool.max_len, 1))[:, None] * 10000.0 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))
        self.table = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
        self.pad, self.apart = pad, apart
        self.pool.upload()
        self.upload()

    def upload(self):
        n, dt, up = self.tokens, self.dt, GpuBuffer.from_bytes
        flat = [x.reshape(n, -1) for x in (self.q, self.k, self.v)]
        if self.apart:
            fill = [np.zeros((n, self.pad), np.float32) for _ in range(3)]
            self.bufs = [up(pack_f32(np.concatenate([x, f], 1), dt)) for x, f in zip(flat, fill)]
            self.at, self.strides = [b.ptr for b in self.bufs], tuple(x.shape[1] + self.pad for x in flat)
        else:
            rows = np.concatenate(flat + [np.zeros((n, self.pad), np.float32)], 1)
            self.bufs = [up(pack_f32(rows, dt))]
            b, e = self.bufs[0].ptr, dt.size_bytes
            self.at, self.strides = [b, b + flat[0].shape[1] * e, b + (flat[0].shape[1] + flat[1].shape[1]) * e], (rows.shape[1],) * 3
        self.tb, self.ob = up(self.table.tobytes()), up(np.array(self.offsets, "<u4").tobytes())
        self.q_out = up(b"\xa5" * (n * self.hq * self.dim * dt.size_bytes))
        self.batch = ops.KvBatch(self.pool.pb, self.pool.width, self.pool.lb, len(self.lens), n, self.pool.max_len, offsets=self.ob)

    def call(self):
        ops.kv_append(self.dt, self.pool.cache, self.batch, self.at[1], self.at[2], row_stride=self.strides, q=self.at[0], q_out=self.q_out, hq=self.hq, cos_sin=self.tb if self.rot else None,
                      n_positions=self.table.shape[0], rot=self.rot, neighbours=self.neighbours)

    def want(self):
        """Queries (None where not written), and the pool's arrays."""
        pool, dt = self.pool, self.dt
        q = np.full(self.q.shape, np.nan, np.float32)
        written = np.zeros(self.tokens, bool)
        for seq, row, place in ref.spans(self.lens, self.offsets, pool.max_len):
            if place < 0:
                continue
            written[row] = True
            at = np.array([place])
            q[row] = typed(ref.turned(self.q[row:row + 1], at, self.table, self.rot, self.neighbours), dt)[0]
            page = pool.pages[seq, place // pool.page]
            if page >= pool.n_pages:
                continue
            for part, x in zip(pool.parts, (ref.turned(self.k[row:row + 1], at, self.table, self.rot, self.neighbours), self.v[row:row + 1])):
                for arr, new in zip(part, ref.quantize(x[0], self.group, dt)):
                    arr[page, :, place % pool.page] = new
        return q, written

    def hold(self):
        q, written = self.want()
        raw = np.frombuffer(self.q_out.read_bytes(), np.uint8).reshape(self.tokens, -1)
        got = unpack_f32(raw.tobytes(), self.dt).reshape(self.q.shape)
        assert np.array_equal(got[written], q[written], equal_nan=True)
        assert np.all(raw[~written] == 0xA5)
        for got, want in zip(self.pool.downloaded(), self.pool.parts):
            for g, w in zip(got, want):
                assert np.array_equal(g, w, equal_nan=True)


CASES = [  # lens, rows, options
    ([1], [1], {}), ([17], [17], dict(group=32)), ([5, 40, 1, 33], [1, 1, 1, 1], dict(hq=8, hkv=8)), ([16, 0, 31], [16, 0, 3], dict(dim=64)), ([100, 64, 3], [70, 64, 2], dict(dim=256, group=128, hkv=1, hq=1)),
    ([50, 20], [50, 5], dict(page=64, neighbours=True)), ([50, 20], [50, 5], dict(rot=64, group=128)), ([50, 20], [50, 5], dict(rot=32, neighbours=True, dim=64, group=32)),
    ([33], [20], dict(rot=20)), ([33], [20], dict(rot=90)), ([33], [20], dict(rot=6, neighbours=True)), ([33], [20], dict(rot=0)), ([9, 3], [9, 3], dict(hq=3, hkv=1, dim=64, pad=8)),
    ([9, 3], [9, 3], dict(hq=6, hkv=3, apart=True, pad=16)), ([9, 3], [4, 3], dict(gaps=True)), ([4, 0, 2], [6, 1, 2], {}), ([90], [8], dict(max_len=77)), ([300] * 70, [1] * 70, dict(hq=2, hkv=1, dim=64)),
    ([2, 3] * 2100, [1, 0] * 2100, dict(hq=1, hkv=1, dim=64))]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,rows,more", CASES, ids=lambda v: str(v).replace(" ", "")[:40])
def test_append(dt, lens, rows, more):
    print(f"[case] kv_append {dt.name} {str(lens)[:40]} {str(rows)[:40]} {more}", flush=True)
    c = Append(dt, lens, rows, **more)
    c.call()
    c.hold()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("more", [dict(), dict(neighbours=True), dict(rot=40), dict(dim=256, rot=96)], ids=str)
def test_queries_in_place(dt, more):
    c = Append(dt, [40, 7], [30, 7], hq=6, hkv=2, **more)
    q = c.at[0]
    ops.kv_append(dt, c.pool.cache, c.batch, c.at[1], c.at[2], row_stride=c.strides, q=q, q_out=q, q_out_stride=c.strides[0], hq=c.hq, cos_sin=c.tb, n_positions=c.table.shape[0], rot=c.rot,
                  neighbours=c.neighbours)
    want, _ = c.want()
    got = unpack_f32(c.bufs[0].read_bytes(), dt).reshape(c.tokens, -1)
    n = c.hq * c.dim
    assert np.array_equal(got[:, :n].reshape(want.shape), want)
    assert np.array_equal(got[:, n:], np.concatenate([c.k.reshape(c.tokens, -1), c.v.reshape(c.tokens, -1)], 1))


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_no_queries_and_equal_rows(dt):
    """Without queries, and with offsets None: 2 rows each."""
    c = Append(dt, [12, 2, 30], [2, 2, 2])
    batch = ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 3, 6, c.pool.max_len)
    ops.kv_append(dt, c.pool.cache, batch, c.at[1], c.at[2], row_stride=c.strides, cos_sin=c.tb, n_positions=c.table.shape[0], rot=c.rot)
    c.want()
    for got, want in zip(c.pool.downloaded(), c.pool.parts):
        for g, w in zip(got, want):
            assert np.array_equal(g, w, equal_nan=True)
    assert c.q_out.read_bytes() == b"\xa5" * c.q_out.nbytes


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_pages_that_are_none(dt):
    """Tokens on no page are not stored (nor read), their queries are turned all the same."""
    c = Append(dt, [40, 20], [40, 20])
    c.pool.pages[0, 1], c.pool.pages[1, 0] = c.pool.n_pages, ref.NO_PAGE
    c.pool.pb.upload(c.pool.pages.astype("<u4").tobytes())
    c.call()
    c.hold()
    _read_holds(c)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
def test_no_numbers(dt, bad):
    """A group with a NaN or an infinity reads as NaN, all of it, and nothing else does; queries have what the turn makes of them."""
    c = Append(dt, [20], [20], rot=64, group=32)
    c.q[3, 1, 5], c.k[2, 0, 100], c.v[5, 1, 0] = bad, bad, bad
    c.upload()
    c.call()
    c.hold()
    _read_holds(c)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
def test_groups_of_one_value_and_of_the_smallest_steps(dt):
    c = Append(dt, [6], [6], rot=0)
    c.v[0] = 0
    c.v[1] = -3.5
    c.v[2, :, ::2], c.v[2, :, 1::2] = 1.0, 1.0 + 2.0 ** -7
    c.v[3] *= 1e-6
    c.v[4, 0, 0] = 60000
    c.v = typed(c.v, dt)
    c.upload()
    c.call()
    c.hold()
    _read_holds(c)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_a_page_is_what_the_packed_format_is(dt, group):
    """Values that are not turned are stored to the bit as affine_quantize packs them."""
    hkv, dim, page = 3, 128, 16
    c = Append(dt, [page], [page], hkv=hkv, dim=dim, group=group, page=page, rot=0)
    c.call()
    at = int(c.pool.pages[0, 0])
    x = c.v.swapaxes(0, 1)   # [head, place, dim]: a page
    xb, wb, sb, bb = GpuBuffer.from_bytes(pack_f32(x, dt)), GpuBuffer(x.size // 2), GpuBuffer(x.size // group * dt.size_bytes), GpuBuffer(x.size // group * dt.size_bytes)
    ops.affine_quantize(dt, 4, group, xb, wb, sb, bb, x.size)
    for buf, mine in zip((wb, sb, bb), c.pool.bufs[3:]):
        got = buf.read_bytes()
        assert mine.read_bytes()[at * len(got):(at + 1) * len(got)] == got


def _read_holds(c):
    pool, dt = c.pool, c.dt
    size = c.tokens * pool.hkv * pool.dim * dt.size_bytes
    outs = [GpuBuffer.from_bytes(b"\xa5" * size) for _ in range(2)]
    ops.kv_read(dt, pool.cache, c.batch, *outs)
    raw = [np.frombuffer(o.read_bytes(), np.uint8).reshape(c.tokens, -1) for o in outs]
    got = [unpack_f32(r.tobytes(), dt).reshape(c.tokens, pool.hkv, pool.dim) for r in raw]
    written = np.zeros(c.tokens, bool)
    f = np.float32
    with np.errstate(all="ignore"):
        for seq, row, place in ref.spans(c.lens, c.offsets, pool.max_len):
            if place < 0 or pool.pages[seq, place // pool.page] >= pool.n_pages:
                continue
            written[row] = True
            for g, (codes, scales, biases) in zip(got, pool.parts):
                at = pool.pages[seq, place // pool.page], slice(None), place % pool.page
                s, b = (np.repeat(x[at], pool.group, -1) for x in (scales, biases))
                assert np.array_equal(g[row], typed((s * codes[at].astype(f)).astype(f) + b, dt), equal_nan=True)
    for r in raw:
        assert np.all(r[~written] == 0xA5)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,rows,more", CASES, ids=lambda v: str(v).replace(" ", "")[:40])
def test_read(dt, lens, rows, more):
    print(f"[case] kv_read {dt.name} {str(lens)[:40]} {str(rows)[:40]} {more}", flush=True)
    _read_holds(Append(dt, lens, rows, **more))


def test_one_of_the_two():
    c = Append(DType.BF16, [20], [20])
    size = c.tokens * 2 * 128 * 2
    both = [GpuBuffer(size) for _ in range(2)]
    ops.kv_read(c.dt, c.pool.cache, c.batch, *both)
    for i in range(2):
        one = GpuBuffer(size)
        ops.kv_read(c.dt, c.pool.cache, c.batch, *((one, None) if i == 0 else (None, one)))
        assert one.read_bytes() == both[i].read_bytes()


def test_captured():
    """A captured append and read follow lens, offsets and pages as they are when it is replayed."""
    c = Append(DType.BF16, [40, 20, 0], [1, 1, 1])
    out = [GpuBuffer(3 * 2 * 128 * 2) for _ in range(2)]
    g = Graph()
    try:
        with g:
            c.call()
            ops.kv_read(c.dt, c.pool.cache, c.batch, *out)
        assert g.nodes == 2
        for turn in range(4):
            c.q, c.k, c.v = (typed(c.rng.standard_normal(x.shape), c.dt) for x in (c.q, c.k, c.v))
            c.bufs[0].upload(pack_f32(np.concatenate([x.reshape(3, -1) for x in (c.q, c.k, c.v)], 1), c.dt))
            c.lens = c.pool.lens = [40 + turn, 20 + 3 * turn, turn if turn != 2 else 0]
            c.pool.lb.upload(np.array(c.lens, "<u4").tobytes())
            c.pool.pages[2, 0] = c.pool.spare[0] if turn > 1 else ref.NO_PAGE
            c.pool.pb.upload(c.pool.pages.astype("<u4").tobytes())
            c.q_out.upload(b"\xa5" * c.q_out.nbytes)
            g.replay()
            c.hold()
            got = [o.read_bytes() for o in out]
            ops.kv_read(c.dt, c.pool.cache, c.batch, *out)
            ops.sync()
            assert [o.read_bytes() for o in out] == got
    finally:
        g.close()


def test_refusals():
    c = Append(DType.BF16, [20], [4])
    dt, cache, batch = c.dt, c.pool.cache, c.batch
    good = dict(row_stride=c.strides, q=c.at[0], q_out=c.q_out, hq=c.hq, cos_sin=c.tb, n_positions=c.table.shape[0], rot=c.rot)
    before = [b.read_bytes() for b in c.pool.bufs]

    def refused(code, k=c.at[1], v=c.at[2], dt=dt, cache=cache, batch=batch, **more):
        with pytest.raises(MtqError) as e:
            ops.kv_append(dt, cache, batch, k, v, **{**good, **more})
        assert e.value.code == code

    def other(**more):
        o = ops.KvCache(*c.pool.bufs, c.pool.n_pages, 16, 2, 128, 64)
        for k, v in more.items():
            setattr(o, k, v)
        return o

    refused(-2, k=None)
    refused(-2, v=None)
    refused(-2, q=None)
    refused(-2, q_out=None)
    refused(-2, cos_sin=None)
    refused(-2, k=c.at[1] + 2)
    refused(-2, q_out=c.q_out.ptr + 8)
    refused(-2, cos_sin=c.tb.ptr + 4)
    refused(-2, row_stride=c.strides[0] + 1)
    refused(-3, row_stride=64)
    refused(-2, q_out=c.at[0])                       # (in place with another stride)
    refused(-3, rot=130)
    refused(-3, rot=7)
    refused(-3, n_positions=c.pool.max_len - 1)
    refused(-2, dt=3)
    refused(-3, cache=other(page_size=24))
    refused(-3, cache=other(page_size=8))
    refused(-3, cache=other(group_size=16))
    refused(-3, cache=other(head_dim=64, group_size=128))
    refused(-7, cache=other(head_dim=96))
    refused(-3, cache=other(n_heads=0))
    refused(-2, cache=other(v_scales=None))
    refused(-2, cache=other(k_codes=c.pool.bufs[0].ptr + 4))
    refused(-3, batch=ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 1, 4, c.pool.width * 16 + 1, offsets=c.ob))
    refused(-3, batch=ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 3, 4, 16))
    refused(-3, batch=ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 1, 1 << 24, 16, offsets=c.ob))
    with pytest.raises(MtqError):
        ops.kv_read(dt, cache, batch, c.q_out.ptr + 2, None)
    assert [b.read_bytes() for b in c.pool.bufs] == before
    # Nothing to do is no error, whatever the buffers.
    none = ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 1, 0, 16)
    ops.kv_append(dt, cache, none, None, None)
    ops.kv_read(dt, cache, none, None, None)
    ops.kv_read(dt, cache, batch, None, None)
