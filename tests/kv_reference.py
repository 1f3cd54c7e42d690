"""A paged cache in packed 4-bit codes on the host, and its operators from their definitions: codes to the bit in f32 steps, attention in 64 bits."""
import numpy as np

from metaltile_amd import DType, GpuBuffer, ops, pack_f32, unpack_f32

DTYPES = [DType.F32, DType.F16, DType.BF16]
HALF_STEP = {DType.F32: 2.0 ** -24, DType.F16: 2.0 ** -11, DType.BF16: 2.0 ** -8}
NO_PAGE = 0xFFFFFFFF


def typed(x, dt):
    return unpack_f32(pack_f32(np.asarray(x, np.float32), dt), dt).reshape(np.shape(x))


def quantize(x, group, dt):
    """Codes u8[..., dim], scales and biases (in T, as f32) [..., dim / group] of f32 values: each step rounded to f32. A group with a NaN or an infinity: NaN."""
    f = np.float32
    x = np.asarray(x, f)
    g = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        fine = np.isfinite(g).all(-1)
        low, top = g.min(-1), g.max(-1)
        scale = ((top - low) / f(15)).astype(f)
        scale = np.where(scale < f(1e-7), f(1), scale)
        inv = (f(1) / scale).astype(f)
        q = ((g - low[..., None]).astype(f) * inv[..., None]).astype(f) + f(0.5)
        codes = np.where(fine[..., None], np.clip(q, 0, 15), 0).astype(np.uint8)
        scale, low = np.where(fine, scale, np.nan).astype(f), np.where(fine, low, np.nan).astype(f)
        return codes.reshape(x.shape), typed(scale, dt), typed(low, dt)


def words(codes):
    return (codes.astype(np.uint32).reshape(*codes.shape[:-1], -1, 8) << np.arange(0, 32, 4, dtype=np.uint32)).sum(-1).astype("<u4")


def codes_of(w):
    return (w[..., None] >> np.arange(0, 32, 4, dtype=np.uint32) & 15).reshape(*w.shape[:-1], -1).astype(np.uint8)


def turned(x, places, table, rot, neighbours):
    """x f32[tokens, heads, dim] turned by the table's rows: products and sums rounded to f32."""
    f = np.float32
    out = np.array(x, f)
    if rot:
        c, s = table[places][:, None, :rot // 2], table[places][:, None, rot // 2:]
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if neighbours else (x[..., :rot // 2], x[..., rot // 2:rot])
        with np.errstate(all="ignore"):
            one, two = (a * c).astype(f) - (b * s).astype(f), (b * c).astype(f) + (a * s).astype(f)
        if neighbours:
            out[..., 0:rot:2], out[..., 1:rot:2] = one, two
        else:
            out[..., :rot // 2], out[..., rot // 2:rot] = one, two
    return out


class Pool:
    """Pages of random codes, scales and biases. `rough`: NaN and the largest scales where no token is."""

    def __init__(self, dt, rng, lens, hkv, dim, group, page, spare=2, width=None, max_len=None):
        self.dt, self.hkv, self.dim, self.group, self.page, self.lens = dt, hkv, dim, group, page, list(lens)
        counts = [-(-n // page) for n in lens]
        self.n_pages = sum(counts) + spare
        self.width = max(1, max(counts, default=0)) if width is None else width
        order = rng.permutation(self.n_pages).astype(np.uint32)
        self.pages = np.full((len(lens), self.width), NO_PAGE, np.uint32)
        at = 0
        for i, n in enumerate(counts):
            self.pages[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, hkv, page)
        self.parts = []
        for offset in (1.0, 0.0):   # keys have an offset to each channel
            codes = rng.integers(0, 16, (*shape, dim), dtype=np.uint8)
            scales = typed(0.05 + 0.3 * rng.random((*shape, dim // group)), dt)
            biases = typed(-7.5 * scales + offset * rng.standard_normal((hkv, 1, dim // group)) + 0.3 * rng.standard_normal(scales.shape), dt)
            self.parts.append([codes, scales, biases])
        self.spare = order[at:]
        used = np.zeros((self.n_pages, page), bool)
        for i, n in enumerate(lens):
            for p in range(n):
                used[self.pages[i, p // page], p % page] = True
        for codes, scales, biases in self.parts:
            hidden = ~np.broadcast_to(used[:, None, :, None], scales.shape)
            scales[hidden] = np.where(rng.random(hidden.sum()) < 0.5, np.nan, np.inf)
            biases[hidden] = np.nan
        self.max_len = self.width * page if max_len is None else max_len

    def upload(self):
        self.bufs = []
        for codes, scales, biases in self.parts:
            self.bufs += [GpuBuffer.from_bytes(words(codes).tobytes()), GpuBuffer.from_bytes(pack_f32(scales, self.dt)), GpuBuffer.from_bytes(pack_f32(biases, self.dt))]
        self.cache = ops.KvCache(*self.bufs, self.n_pages, self.page, self.hkv, self.dim, self.group)
        self.pb, self.lb = GpuBuffer.from_bytes(self.pages.astype("<u4").tobytes()), GpuBuffer.from_bytes(np.array(self.lens, "<u4").tobytes())
        return self

    def batch(self, offsets=None, n_tokens=None):
        """offsets: a list, or None with equally many rows each."""
        self.ob = None if offsets is None else GpuBuffer.from_bytes(np.array(offsets, "<u4").tobytes())
        return ops.KvBatch(self.pb, self.width, self.lb, len(self.lens), offsets[-1] if n_tokens is None else n_tokens, self.max_len, offsets=self.ob)

    def downloaded(self):
        """The three arrays of keys and of values, as they are on the device."""
        out = []
        for i in (0, 3):
            shape = (self.n_pages, self.hkv, self.page)
            w = np.frombuffer(self.bufs[i].read_bytes(), "<u4").reshape(*shape, -1)
            out.append([codes_of(w)] + [unpack_f32(self.bufs[i + j].read_bytes(), self.dt).reshape(*shape, -1) for j in (1, 2)])
        return out

    def of(self, seq, n):
        """Of a sequence's first n tokens: which are on a page, and for keys and values (codes - 8) * scale and value, f64[hkv, n, dim]."""
        p = np.arange(n)
        page = self.pages[seq, p // self.page] if n else np.zeros(0, np.uint32)
        there = page < self.n_pages
        page = np.where(there, page, 0)
        out = []
        for codes, scales, biases in self.parts:
            c, s, b = (x[page, :, p % self.page].swapaxes(0, 1).astype(np.float64) for x in (codes, scales, biases))
            s, b = np.repeat(s, self.group, -1), np.repeat(b, self.group, -1)
            with np.errstate(all="ignore"):
                out.append((s * (c - 8), s * c + b))
        return there, out


def spans(lens, offsets, max_len):
    """(sequence, row, place) of every row with its place (negative: none)."""
    for i, n in enumerate(lens):
        n = min(n, max_len)
        rows = offsets[i + 1] - offsets[i]
        for j in range(rows):
            yield i, offsets[i] + j, n - rows + j


def attention(pool, q, offsets, hq, scale, window, dt, rounded=False):
    """(out, tolerance) f64[rows, hq, dim] of q[rows, hq, dim].

    Tolerance. A score is a sum of dim products of q and 16 + code, f32, scaled by group and joined with the bias' share: at most (dim + 24) roundings of 2^-24 of
    scale * sum |q| (48 s + |k|), and a probability's relative error is twice that (its own score's and the largest's) and 2^-19 for exp's
    argument of up to 2^4 in base 2 and its own error. p s is rounded by half a step of what it is held in (bf16 2^-8, 16 bits 2^-16, 24 bits 2^-23) and multiplies
    code - 8. Sums over n tokens are f32, one after the other within a lane of a matrix instruction's row and then over waves and slices: (n / 8 + 128) 2^-24 of the sum of
    magnitudes p (64 s + |v|). At the end half a step of T, and for f16 2^-25 below 2^-14.

    `rounded`: keys, values and weights are in T (sequences of many rows, f16 and bf16). With u half a step of T a key is off by u |k|, a score by u scale sum |q| |k| and
    a probability by e^(2 of the largest of these) - 1; p and v are off by u each, together less than 2.02 u of p |v|; and in f16 a key and a weight (of at least one that is 1)
    below 2^-14 by 2^-25.
    """
    held = {DType.F32: 2.0 ** -23, DType.F16: 2.0 ** -16, DType.BF16: 2.0 ** -8}[dt]
    shared = hq // pool.hkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    cached = {}
    with np.errstate(all="ignore"):
        for seq, row, place in spans(pool.lens, offsets, pool.max_len):
            n = min(pool.lens[seq], pool.max_len)
            if seq not in cached:
                cached[seq] = pool.of(seq, n)
            there, ((kc, k), (vc, v)) = cached[seq]
            lo = max(0, place + 1 - window) if window else 0
            at = np.arange(lo, place + 1)
            at = at[there[at]] if at.size else at
            if at.size == 0:
                continue
            for h in range(hq):
                x, kk, vv = q[row, h].astype(np.float64), k[h // shared][at], v[h // shared][at]
                s = scale * (kk @ x)
                e = np.exp(s - s.max())
                p = e / e.sum()
                o = p @ vv
                step_k, step_v = (_steps(pool, part, seq, h // shared, at) for part in (0, 1))
                size = abs(scale) * ((48 * step_k + np.abs(kk)) @ np.abs(x))
                rel = 2 * (pool.dim + 24) * 2.0 ** -24 * size.max() + 2.0 ** -19
                if rounded:
                    u, least = HALF_STEP[dt], 2.0 ** -25 if dt == DType.F16 else 0.0
                    rel = np.expm1(rel + 2 * (abs(scale) * ((u * np.abs(kk) + least) @ np.abs(x))).max())
                terms = p @ (64 * step_v + np.abs(vv))
                out[row, h] = o
                tol[row, h] = rel * (p @ np.abs(vv) + np.abs(o)) + (2.02 * u * (p @ np.abs(vv)) + at.size * least * (1 + np.abs(vv).max(0)) if rounded else held * (p @ np.abs(vc[h // shared][at]))) + (at.size / 8 + 128) * 2.0 ** -24 * terms \
                    + HALF_STEP[dt] * np.abs(o) + (2.0 ** -25 if dt == DType.F16 else 0)
    return out, tol


def _steps(pool, part, seq, head, at):
    """The largest scale of each token, [tokens, 1]."""
    s = np.abs(pool.parts[part][1][pool.pages[seq, at // pool.page], head, at % pool.page].astype(np.float64))
    return np.where(np.isnan(s), 0, s).max(-1, keepdims=True)
