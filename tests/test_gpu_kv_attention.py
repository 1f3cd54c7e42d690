"""Attention over the paged 4-bit cache against 64 bits; the tolerance is derived in kv_reference.attention. Memory where no token is holds NaN and infinities."""
import ctypes as C

import numpy as np
import pytest

from metaltile_amd import DType, GpuBuffer, MtqError, _lib, ops, pack_f32, unpack_f32
from metaltile_amd.runtime import _ensure_init
from tests import kv_reference as ref
from tests.hip_graph import Graph
from tests.kv_reference import DTYPES, typed

pytestmark = pytest.mark.gpu


class Attention:
    def __init__(self, dt, lens, rows, hq=4, hkv=2, dim=128, group=64, page=16, window=0, seed=1, pad=0, gaps=False, max_len=None, width=None, scale=None, equal=False):
        self.dt, self.lens, self.hq, self.dim, self.window = dt, lens, hq, dim, window
        rng = self.rng = np.random.default_rng(seed)
        self.pool = ref.Pool(dt, rng, lens, hkv, dim, group, page, max_len=max_len, width=width).upload()
        self.offsets = np.concatenate([[0], np.cumsum(rows)]).astype(int).tolist()
        if gaps:
            self.offsets = [o + 3 for o in self.offsets]
        self.tokens = n = self.offsets[-1] + (2 if gaps else 0)
        self.scale = dim ** -0.5 if scale is None else scale
        self.q = typed(rng.standard_normal((n, hq, dim)), dt)
        self.stride, self.equal = hq * dim + pad, equal
        self.upload()

    def upload(self):
        n, up = self.tokens, GpuBuffer.from_bytes
        rows = np.concatenate([self.q.reshape(n, -1), np.full((n, self.stride - self.hq * self.dim), np.nan, np.float32)], 1)
        self.qb, self.out = up(pack_f32(rows, self.dt)), up(b"\xa5" * (n * self.stride * self.dt.size_bytes))
        self.ob = None if self.equal else up(np.array(self.offsets, "<u4").tobytes())
        self.batch = ops.KvBatch(self.pool.pb, self.pool.width, self.pool.lb, len(self.lens), n, self.pool.max_len, offsets=self.ob)

    def call(self):
        ops.kv_attention(self.dt, self.pool.cache, self.batch, self.qb, self.out, self.hq, self.scale, window=self.window, q_stride=self.stride, out_stride=self.stride)

    def result(self):
        raw = np.frombuffer(self.out.read_bytes(), np.uint8).reshape(self.tokens, -1)
        wide = self.hq * self.dim * self.dt.size_bytes
        rest = np.concatenate([raw[:, wide:].ravel(), raw[:self.offsets[0]].ravel(), raw[self.offsets[-1]:].ravel()])
        assert np.all(rest == 0xA5)   # between rows and outside all sequences
        return unpack_f32(raw[:, :wide].tobytes(), self.dt).reshape(self.tokens, self.hq, self.dim)

    def rounded(self, kernel=0):
        """Whether keys and values are rounded to T: in the kernel for prompts, of 16-bit types."""
        return self.dt != DType.F32 and (kernel == 4 or kernel == 0 and self.tokens * (self.hq // self.pool.hkv) > 64 * len(self.pool.lens))   # (of calls that do not fill the card)

    def hold(self, kernel=0):
        got = self.result()[self.offsets[0]:self.offsets[-1]]
        want, tol = (x[self.offsets[0]:self.offsets[-1]] for x in ref.attention(self.pool, self.q, self.offsets, self.hq, self.scale, self.window, self.dt, self.rounded(kernel)))
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        far = np.abs(got - want)[fine] / np.maximum(tol[fine], 1e-30)
        assert np.all(far <= 1), f"{far.max()} of the tolerance"


CASES = [  # lens, rows, options
    ([1], [1], {}), ([2], [2], {}), ([15], [1], {}), ([16], [1], {}), ([17], [1], {}), ([31], [3], {}), ([33], [1], dict(hq=1, hkv=1)), ([100], [1], dict(hq=8, hkv=1)), ([257], [1], dict(hq=16, hkv=1)),
    ([300], [1], dict(hq=40, hkv=2)), ([513, 5, 64, 1], [1, 1, 1, 1], dict(hq=6, hkv=2)), ([700], [2], dict(dim=64, group=32)), ([700], [3], dict(dim=64, group=64, page=64)),
    ([700], [1], dict(dim=256, group=32)), ([300], [4], dict(dim=256, group=128)), ([300, 0, 40], [5, 1, 2], dict(dim=256, group=64, hq=2, hkv=1)), ([400], [1], dict(group=32)), ([400], [1], dict(group=128)),
    ([64, 30], [64, 30], {}), ([200], [200], dict(group=32, hq=3, hkv=1)), ([200], [77], dict(group=128, hq=2, hkv=2)), ([130, 1, 0, 65], [130, 1, 0, 20], dict(dim=64)), ([150], [150], dict(dim=256, hq=2, hkv=1)),
    ([150, 90], [50, 90], dict(dim=256, group=128, page=128, hq=4, hkv=1)), ([90, 20], [8, 3], dict(gaps=True, pad=8)), ([100, 60], [100, 60], dict(gaps=True, pad=16)),
    ([4, 0, 2], [6, 1, 2], {}), ([20, 0, 2], [60, 33, 2], {}), ([90], [8], dict(max_len=77)), ([90], [60], dict(max_len=77)), ([40, 300], [2, 2], dict(equal=True)), ([40, 300], [40, 40], dict(equal=True)),
    ([500], [1], dict(window=1)), ([500], [1], dict(window=100)), ([500, 20], [9, 9], dict(window=33)), ([300], [200], dict(window=17)), ([300, 70], [200, 70], dict(window=64, dim=64)),
    ([300], [1], dict(scale=3.0)), ([200], [100], dict(scale=3.0)), ([300], [1], dict(scale=0.0)), ([300], [2], dict(scale=-0.1)), ([1500], [1], dict(hq=2, hkv=1)), ([1500, 3], [30, 3], dict(hq=2, hkv=1)),
    ([(7 * i) % 50 for i in range(150)], [i % 2 for i in range(150)], dict(hq=2, hkv=1, dim=64)), ([(7 * i) % 50 for i in range(150)], [(i * 5) % 7 for i in range(150)], dict(hq=2, hkv=1, dim=64))]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,rows,more", CASES, ids=lambda v: str(v).replace(" ", "")[:40])
def test_attention(dt, lens, rows, more):
    print(f"[case] kv_attention {dt.name} {str(lens)[:40]} {str(rows)[:40]} {more}", flush=True)
    c = Attention(dt, lens, rows, **more)
    c.call()
    c.hold()


@pytest.fixture
def option():
    lib, used = _ensure_init(), set()

    def put(name, value):
        used.add(name)
        _lib.check(lib.mtq_set_option(name.encode(), value))

    yield put
    for name in used:
        _lib.check(lib.mtq_set_option(name.encode(), 0))


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,rows,more", CASES, ids=lambda v: str(v).replace(" ", "")[:40])
def test_either_kernel(dt, lens, rows, more, option):
    """Whatever the sizes: the kernel for few rows, the ones for many, the one for up to four, in one slice and in several."""
    print(f"[case] kv_attention {dt.name} {str(lens)[:40]} {str(rows)[:40]} {more}, all kernels", flush=True)
    c = Attention(dt, lens, rows, **more)
    for kernel, slices in ((1, 1), (1, 3), (2, 1), (2, 5), (3, 1), (3, 4), (4, 1), (4, 3)):
        option("kv.kernel", kernel)
        option("kv.slices", slices)
        c.out.upload(b"\xa5" * c.out.nbytes)
        c.call()
        c.hold(kernel)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_every_head(dt, dim, group):
    for lens, rows in (([330, 70], [1, 2]), ([330, 70], [100, 70])):
        c = Attention(dt, lens, rows, dim=dim, group=group, hq=6, hkv=2)
        c.call()
        c.hold()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,kernel", [([1, 1], 0), ([200, 40], 0), ([200, 40], 4)], ids=str)
def test_pages_that_are_none(dt, rows, kernel, option):
    """Tokens on no page do not count; a sequence that is on none is zeros."""
    c = Attention(dt, [220, 40], rows)
    c.pool.pages[0, [0, 3, 4, 9]], c.pool.pages[1] = c.pool.n_pages, ref.NO_PAGE
    c.pool.pb.upload(c.pool.pages.astype("<u4").tobytes())
    option("kv.kernel", kernel)
    c.call()
    c.hold(kernel)
    assert np.all(c.result()[c.offsets[1]:] == 0)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,kernel", [([3, 1], 0), ([3, 1], 1), ([130, 40], 0), ([130, 40], 4)], ids=str)
@pytest.mark.parametrize("what", ["q", "k_scale", "k_bias", "v_scale", "v_bias"])
@pytest.mark.parametrize("window", [0, 20])
def test_no_numbers(dt, rows, kernel, what, window, option):
    """A NaN reaches the rows that see it, and of a value's only its group; none of the others."""
    c = Attention(dt, [140, 40], rows, window=window, dim=128, group=64)
    pool = c.pool
    if what == "q":
        c.q[1, 2, 5] = np.nan
        c.upload()
    else:
        arr = pool.parts[what[0] == "v"][1 if "scale" in what else 2]
        for place in (138, 100, 77, 31):
            arr[pool.pages[0, place // 16], 1, place % 16, 1] = np.nan
        for i, (codes, scales, biases) in enumerate(pool.parts):
            pool.bufs[3 * i + 1].upload(pack_f32(scales, dt))
            pool.bufs[3 * i + 2].upload(pack_f32(biases, dt))
    option("kv.kernel", kernel)
    c.call()
    c.hold(kernel)
    got = c.result()
    assert np.isnan(got).any() and not np.isnan(got).all()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("rows,kernel", [([1], 0), ([1], 1), ([100], 0), ([100], 4)], ids=str)
def test_scores_far_apart(dt, rows, kernel, option):
    """Scores of thousands: one token takes it all, wherever it is, and nothing passes the exponent."""
    option("kv.kernel", kernel)
    for place in (0, 31, 32, 170):
        c = Attention(dt, [200], rows, hq=2, hkv=1, scale=1.0, seed=place + 2)
        codes, scales, biases = c.pool.parts[0]
        at = c.pool.pages[0, place // 16], 0, place % 16
        scales[at], biases[at] = 100.0, -750.0
        for i, x in ((1, scales), (2, biases)):
            c.pool.bufs[i].upload(pack_f32(x, dt))
        c.call()
        got = c.result()
        want, tol = ref.attention(c.pool, c.q, c.offsets, c.hq, c.scale, 0, dt)
        assert np.all(np.isfinite(got))
        # The scores' own rounding is past what a tolerance says anything about where several are near the largest: rows with one far ahead are held.
        kk = c.pool.of(0, 200)[1][0][1][0]
        for row in range(c.tokens):
            n = 200 - c.tokens + row + 1
            for h in range(2):
                s = np.sort(kk[:n] @ c.q[row, h].astype(np.float64))
                if n == 1 or s[-1] - s[-2] > 60:
                    assert np.all(np.abs(got[row, h] - want[row, h]) <= HELD[dt] * (np.abs(want[row, h]) + 8 * 0.4))


HELD = {DType.F32: 2.0 ** -18, DType.F16: 2.0 ** -10, DType.BF16: 2.0 ** -6}   # (a rounding of p s, whose codes are up to 8 steps of 0.35 from the middle, and one of the result)


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("lens,rows", [([900, 40], [1, 1]), ([900, 40], [60, 40])], ids=str)
def test_without_scratch(dt, lens, rows):
    c = Attention(dt, lens, rows)
    lib = _ensure_init()
    try:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 1))
        c.call()
        c.hold()
    finally:
        _lib.check(lib.mtq_set_option(b"scratch.most_kb", 0))


def test_the_same_bits_again():
    for rows in ([1, 1, 1], [90, 1, 40]):
        c = Attention(DType.BF16, [1000, 5, 300], rows, hq=8, hkv=2)
        c.call()
        first = c.out.read_bytes()
        for _ in range(3):
            c.out.upload(b"\xa5" * c.out.nbytes)
            c.call()
            assert c.out.read_bytes() == first


@pytest.mark.parametrize("rows,kernel", [([1, 1, 1], 0), ([40, 1, 60], 0), ([40, 1, 60], 4)], ids=str)
def test_captured(rows, kernel, option):
    """A captured call follows lens, pages and queries as they are when it is replayed, other calls with the same scratch between."""
    option("kv.kernel", kernel)
    c = Attention(DType.BF16, [200, 90, 300], rows, hq=8, hkv=2, width=32)
    other = Attention(DType.F16, [1200], [1], hq=16, hkv=2, seed=9)
    other.call()
    g = Graph()
    try:
        with g:
            c.call()
        for turn in range(4):
            c.lens = c.pool.lens = [200 - 3 * turn, 90 - turn, 300 - 50 * turn]
            c.pool.lb.upload(np.array(c.lens, "<u4").tobytes())
            c.q = typed(c.rng.standard_normal(c.q.shape), c.dt)
            c.qb.upload(pack_f32(c.q, c.dt))
            c.out.upload(b"\xa5" * c.out.nbytes)
            g.replay()
            c.hold(kernel)
            got = c.out.read_bytes()
            other.out.upload(b"\xa5" * other.out.nbytes)
            other.call()
            other.hold(kernel)
            c.call()
            ops.sync()
            assert c.out.read_bytes() == got
    finally:
        g.close()


def test_pages_past_32_bits():
    """Codes past 4 GiB of each array, and tokens behind 2^32 elements."""
    hkv, dim, group, page = 8, 128, 64, 256
    n_pages = 40000   # 40000 x 8 x 256 x 64 bytes: 5.2 GB of codes, 328 M scales
    rng = np.random.default_rng(4)
    near = Attention(DType.BF16, [300, 20], [2, 1], hq=16, hkv=hkv, dim=dim, group=group, page=page)
    sizes = [n_pages * hkv * page * dim // 2] + [n_pages * hkv * page * (dim // group) * 2] * 2
    bufs = [GpuBuffer(n) for n in sizes * 2]
    far = np.array(near.pool.pages)
    take = rng.permutation(np.arange(n_pages - 8, n_pages))
    lib = _ensure_init()
    for old, new in zip(np.unique(near.pool.pages[near.pool.pages < near.pool.n_pages]), take):
        far[near.pool.pages == old] = new
        for i, (codes, scales, biases) in enumerate(near.pool.parts):
            for j, data in enumerate((ref.words(codes[old]).tobytes(), pack_f32(scales[old], DType.BF16), pack_f32(biases[old], DType.BF16))):
                arr = np.frombuffer(data, np.uint8)
                _lib.check(lib.mtq_upload(bufs[3 * i + j].ptr + int(new) * arr.nbytes, arr.ctypes.data_as(C.c_void_p), arr.nbytes))
    near.call()
    near.hold()
    want = near.out.read_bytes()
    near.pool.pb.upload(far.astype("<u4").tobytes())
    near.pool.cache = ops.KvCache(*bufs, n_pages, page, hkv, dim, group)
    near.out.upload(b"\xa5" * near.out.nbytes)
    near.call()
    assert near.out.read_bytes() == want
    for b in bufs:
        b.free()


@pytest.mark.parametrize("kernel", [1, 2, 3, 4])
@pytest.mark.parametrize("seqs,longest,window", [(130, 400, 0), (130, 400, 90), (512, 60, 0), (600, 60, 0)])
def test_many_sequences(seqs, longest, window, kernel, option):
    """More sequences than a wave has lanes, than are cut, some without rows and some without tokens: pieces of every length."""
    print(f"[case] kv_attention {seqs} sequences, kernel {kernel}", flush=True)
    rng = np.random.default_rng(seqs)
    lens = [int(n) for n in rng.integers(0, longest, seqs)]
    c = Attention(DType.BF16, lens, [int(n) for n in rng.integers(0, 3, seqs)], hq=2, hkv=1, window=window)
    option("kv.kernel", kernel)
    for slices in (0, 1, 4, 30):
        option("kv.slices", slices)
        c.out.upload(b"\xa5" * c.out.nbytes)
        c.call()
        c.hold(kernel)


@pytest.mark.parametrize("kernel", [0, 1, 3])
@pytest.mark.parametrize("hq", [1, 3, 4, 24])
def test_prompts_among_tokens(kernel, hq, option):
    """Single tokens with a prompt or two among them, in the kernels for few rows: as many sets of rows as a sequence needs, whatever the number of query heads."""
    rng = np.random.default_rng(hq)
    lens = [int(n) for n in rng.integers(1, 200, 70)]
    rows = [1] * 70
    rows[13], rows[69], rows[0], rows[40] = min(lens[13], 90), min(lens[69], 40), 0, 3
    c = Attention(DType.BF16, lens, rows, hq=hq, hkv=1)
    option("kv.kernel", kernel)
    for slices in (0, 1, 3):
        option("kv.slices", slices)
        c.out.upload(b"\xa5" * c.out.nbytes)
        c.call()
        c.hold(kernel)


@pytest.mark.parametrize("kernel", [1, 2, 3, 4])
def test_shared_pages(kernel, option):
    """Sequences whose first pages are the same ones."""
    c = Attention(DType.F16, [200, 180, 90], [3, 40, 20])
    c.pool.pages[1, :8] = c.pool.pages[0, :8]
    c.pool.pages[2, :4] = c.pool.pages[0, :4]
    c.pool.pb.upload(c.pool.pages.astype("<u4").tobytes())
    option("kv.kernel", kernel)
    c.call()
    c.hold(kernel)


@pytest.mark.parametrize("kernel", [1, 2, 3, 4])
def test_a_callers_stream(kernel, option):
    """Queries copied on the caller's stream, the call behind them, and the result back: no wait in between."""
    hip = C.CDLL("libamdhip64.so")
    stream, lib = C.c_void_p(), _ensure_init()
    c = Attention(DType.BF16, [900, 300], [70, 30], hq=4, hkv=2)
    option("kv.kernel", kernel)
    option("kv.slices", 3)
    q, got = c.qb.read_bytes(), np.zeros(c.out.nbytes, np.uint8)
    c.qb.upload(b"\0" * c.qb.nbytes)
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    try:
        _lib.check(lib.mtq_set_stream(stream))
        assert hip.hipMemcpyAsync(C.c_void_p(c.qb.ptr), q, C.c_size_t(len(q)), 1, stream) == 0
        c.call()
        assert hip.hipMemcpyAsync(got.ctypes.data_as(C.c_void_p), C.c_void_p(c.out.ptr), C.c_size_t(got.nbytes), 2, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
    finally:
        _lib.check(lib.mtq_set_stream(None))
        hip.hipStreamDestroy(stream)
    c.hold(kernel)
    assert got.tobytes() == c.out.read_bytes()


def test_a_pool_past_32_bits_of_tokens():
    c = Attention(DType.BF16, [20], [4])
    with pytest.raises(MtqError) as e:
        ops.kv_attention(c.dt, ops.KvCache(*c.pool.bufs, 1 << 27, 16, 2, 128, 64), c.batch, c.qb, c.out, 4, 1.0)
    assert e.value.code == -3 and c.out.read_bytes() == b"\xa5" * c.out.nbytes


def test_refusals():
    c = Attention(DType.BF16, [20], [4])
    dt, cache, batch = c.dt, c.pool.cache, c.batch

    def refused(code, dt=dt, cache=cache, batch=batch, q=c.qb, out=c.out, hq=4, **more):
        with pytest.raises(MtqError) as e:
            ops.kv_attention(dt, cache, batch, q, out, hq, 1.0, **more)
        assert e.value.code == code

    refused(-2, q=None)
    refused(-2, out=None)
    refused(-2, dt=4)
    refused(-2, q=c.qb.ptr + 4)
    refused(-2, out=c.out.ptr + 8)
    for scale in (np.nan, np.inf, -np.inf):
        with pytest.raises(MtqError) as e:
            ops.kv_attention(dt, cache, batch, c.qb, c.out, 4, scale)
        assert e.value.code == -2
    refused(-3, hq=0)
    refused(-3, hq=3)
    refused(-3, q_stride=128)
    refused(-2, out_stride=4 * 128 + 4)
    refused(-3, batch=ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 1, 4, c.pool.width * 16 + 1, offsets=c.ob))
    refused(-7, cache=ops.KvCache(*c.pool.bufs, c.pool.n_pages, 16, 2, 96, 32))
    refused(-3, cache=ops.KvCache(*c.pool.bufs, c.pool.n_pages, 17, 2, 128, 32))
    assert c.out.read_bytes() == b"\xa5" * c.out.nbytes
    ops.kv_attention(dt, cache, ops.KvBatch(c.pool.pb, c.pool.width, c.pool.lb, 1, 0, 16), None, None, 4, 1.0)
