// Writer and reader of a paged cache in packed 4-bit codes (kv_cache.h): memory bounds both, eight values a lane, 16 bytes of 16-bit elements
// on one side and a word of codes on the other.
#include "kv_cache.h"

// Every a*b+c here is two rounded operations, as the packed format's quantiser has them: a code is the same wherever it is made.
#pragma STDC FP_CONTRACT OFF

namespace mtq {

namespace {

// Eight values to p + i; PAST: past the caches. What a large call writes would push out of them what it still reads: 60000 tokens of 8 heads of 64 in f16 are
// read in 34.7 us (4.8 TB/s) so and in 50.2 otherwise, 9300 tokens of 24 heads of 128 appended and read in 33.4 and 42.8. A small call's rows are read next.
template <int DT, bool PAST> __device__ __forceinline__ void kv_store8(void* p, uint64_t i, const float (&v)[8]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    auto put = [](void* to, u32x4 w) {
        if constexpr (PAST) __builtin_nontemporal_store(w, (u32x4*)to);
        else *(u32x4*)to = w;
    };
    if constexpr (DT == DT_F32) {
        put((float*)p + i, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
        put((float*)p + i + 4, u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
    } else {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t)f32_to_elem_bits<DT>(v[2 * j]) | (uint32_t)f32_to_elem_bits<DT>(v[2 * j + 1]) << 16;
        put((uint16_t*)p + i, w);
    }
}

// Eight values as they come from memory.
template <int DT> struct KvRaw {
    uint4 w[DT == DT_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* p, uint64_t i) {
        const uint4* from = (const uint4*)((const uint8_t*)p + i * (DT == DT_F32 ? 4 : 2));
        w[0] = from[0];
        if constexpr (DT == DT_F32) w[1] = from[1];
    }
    __device__ __forceinline__ float operator()(int j) const {
        const uint4& q = w[DT == DT_F32 ? j / 4 : 0];
        const uint32_t d = DT == DT_F32 ? j % 4 : j / 2, x = d == 0 ? q.x : d == 1 ? q.y : d == 2 ? q.z : q.w;
        if constexpr (DT == DT_F32) return __uint_as_float(x);
        else return DT == DT_BF16 ? bf16_bits_to_f32(j & 1 ? x >> 16 : x & 0xFFFFu) : f16_bits_to_f32(j & 1 ? x >> 16 : x & 0xFFFFu);
    }
};
// How pairs lie: none is turned; neighbours, or halves, whose table entries eight values have side by side (multiples of eight, and of sixteen, are turned); any.
enum { KV_PLAIN, KV_NEIGHBOURS, KV_HALVES, KV_ANY };

// Values e0 .. e0 + 7 of a head at p + i: asked for, and then turned by the table's row.
template <int DT, int PAIRS> struct KvTurned {
    KvRaw<DT> own, other;
    KvRaw<DT_F32> c, s;
    __device__ __forceinline__ void load(const KvAppendArgs& a, const void* p, uint64_t i, uint32_t e0, uint32_t place, bool turn) {
        own.load(p, i + e0);
        if (PAIRS == KV_PLAIN || PAIRS == KV_ANY || !turn || e0 >= a.rot) return;
        const uint32_t half = a.rot / 2, j0 = e0 >= half ? e0 - half : e0;
        const float* row = a.cos_sin + (uint64_t)place * a.rot;
        if constexpr (PAIRS == KV_NEIGHBOURS) {
            c.w[0] = *(const uint4*)(row + e0 / 2);
            s.w[0] = *(const uint4*)(row + half + e0 / 2);
            return;
        }
        other.load(p, i + (e0 >= half ? j0 : e0 + half));
        c.load(row, j0);
        s.load(row, half + j0);
    }
    __device__ __forceinline__ void values(const KvAppendArgs& a, const void* p, uint64_t i, uint32_t e0, uint32_t place, bool turn, float (&v)[8]) const {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = own(j);
        if (PAIRS == KV_PLAIN || !turn || e0 >= a.rot) return;
        const float* row = a.cos_sin + (uint64_t)place * a.rot;
        const uint32_t half = a.rot / 2;
        if constexpr (PAIRS == KV_NEIGHBOURS) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float cs = c(j / 2), sn = s(j / 2), x = v[j], y = v[j + 1];
                const float xc = x * cs, ys = y * sn, yc = y * cs, xs = x * sn;
                v[j] = xc - ys;
                v[j + 1] = yc + xs;
            }
        } else if constexpr (PAIRS == KV_HALVES) {   // (all eight are in one half)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float mine = v[j] * c(j), its = other(j) * s(j);
                v[j] = e0 >= half ? mine + its : mine - its;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t e = e0 + j;
                if (e >= a.rot) continue;
                const bool upper = a.neighbours ? e & 1u : e >= half;
                const uint32_t at = a.neighbours ? e / 2 : upper ? e - half : e;
                const float o = load_elem<DT>(p, i + (a.neighbours ? e ^ 1u : upper ? at : e + half));
                const float mine = v[j] * row[at], its = o * row[half + at];
                v[j] = upper ? mine + its : mine - its;
            }
        }
    }
};

// Where the tokens of rows t0 .. t0 + count - 1 lie, one to a lane: the place in its sequence and the page that it is on. All lanes of a wave call.
struct KvRow {
    int32_t place = -1;            // none: -1
    uint32_t page = 0xFFFFFFFFu;
};
__device__ __forceinline__ KvRow kv_rows(const KvArgs& a, uint32_t t0, uint32_t count) {
    const uint32_t lane = threadIdx.x & 63u, t = t0 + lane;
    uint32_t seq, first, next, len;
    if (a.offsets) {
        // 64 beginnings of sequences and their lengths at once, from the one on that row t0 belongs to; a row's sequence is the last that begins at it or before.
        uint32_t s0 = 0;
        if (a.n_seqs >= 64) {
            const uint32_t c = __builtin_amdgcn_readfirstlane(kv_count_upto(a.offsets, a.n_seqs + 1u, t0));
            s0 = c ? c - 1u : 0u;
        }
        const uint32_t begin = s0 + lane <= a.n_seqs ? a.offsets[s0 + lane] : 0xFFFFFFFFu, length = s0 + lane < a.n_seqs ? a.lens[s0 + lane] : 0u;
        uint32_t upto = 0;
        for (uint32_t j = 0; j < count; j++) {
            const uint32_t c = (uint32_t)__popcll(__ballot(begin <= t0 + j));
            upto = lane == j ? c : upto;
        }
        seq = s0 + upto - 1u;   // (none: behind the last)
        first = (uint32_t)__shfl((int)begin, (int)(upto - 1u), 64);
        next = (uint32_t)__shfl((int)begin, (int)upto, 64);
        len = (uint32_t)__shfl((int)length, (int)(upto - 1u), 64);
        if (upto == 64u) {   // behind those 64
            uint32_t lo = s0 + 63u, hi = a.n_seqs + 1u;   // offsets[lo] <= t, and of the entries from hi on none is
            while (hi - lo > 1u) {
                const uint32_t mid = lo + (hi - lo) / 2u;
                if (a.offsets[mid] <= t) lo = mid; else hi = mid;
            }
            seq = lo;
            first = a.offsets[lo];
            next = lo < a.n_seqs ? a.offsets[lo + 1u] : 0u;
            len = lo < a.n_seqs ? a.lens[lo] : 0u;
        }
        if (upto == 0) seq = a.n_seqs;
    } else {
        const uint32_t per = a.n_tokens / a.n_seqs;
        seq = t / per;
        first = seq * per;
        next = first + per;
        len = seq < a.n_seqs ? a.lens[seq] : 0u;
    }
    KvRow r;
    const uint32_t end = next < a.n_tokens ? next : a.n_tokens;
    if (lane >= count || seq >= a.n_seqs || t < first || t >= end) return r;
    const uint32_t held = len < a.max_len ? len : a.max_len, rows = end - first;
    if (held + (t - first) < rows) return r;   // no place
    r.place = (int32_t)(held + (t - first) - rows);
    r.page = a.pages[(uint64_t)seq * a.pages_stride + ((uint32_t)r.place >> a.page_log2)];
    return r;
}
// A lane's units of eight values: U in turn, of a tile of `per_tile` rows or, where a row has more units than the workgroup, of a part of one row.
struct KvTiles {
    uint32_t units, per_tile, parts, magic;   // of a row; rows of a tile; workgroups of a tile; 2^32 / units, rounded up
};
struct KvUnit {
    uint32_t row, unit;   // row of the tile
};
__device__ __forceinline__ KvUnit kv_unit(const KvTiles& t, uint32_t i) {   // (i < 2^16 and units < 2^16 where there are several rows)
    KvUnit u;
    u.row = t.per_tile == 1 ? 0u : __umulhi(i, t.magic);
    u.unit = i - u.row * t.units;
    return u;
}

// Units are the query heads', then the key heads', then the value heads'. All loads of a workgroup's units are under way before the first is used, and a
// head's lanes are neighbours in a wave: queries may be turned in place.
template <int DT, int PAIRS, int U> __global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, KvTiles tiles) {
#pragma clang fp contract(off)
    const KvArgs& kv = a.kv;
    const uint32_t tile = blockIdx.x / tiles.parts, row0 = tile * tiles.per_tile, from = (blockIdx.x - tile * tiles.parts) * (256 * U);
    const uint32_t count = kv.n_tokens - row0 < tiles.per_tile ? kv.n_tokens - row0 : tiles.per_tile;
    const KvRow rows = kv_rows(kv, row0, count);
    const uint32_t words = kv.dim / 8, words_log2 = (uint32_t)__builtin_ctz(words);
    KvTurned<DT, PAIRS> in[U];
    int32_t places[U];
    uint32_t pages[U];
    // Where a unit's eight values begin.
    auto head_of = [&](uint32_t slot) { return slot < a.hq ? slot : slot < a.hq + kv.hkv ? slot - a.hq : slot - a.hq - kv.hkv; };
    auto base_of = [&](uint32_t slot) { return slot < a.hq ? a.q : slot < a.hq + kv.hkv ? a.k : a.v; };
    auto index_of = [&](uint64_t row, uint32_t slot) { return row * (slot < a.hq ? a.q_stride : slot < a.hq + kv.hkv ? a.k_stride : a.v_stride) + (uint64_t)head_of(slot) * kv.dim; };
#pragma unroll
    for (int j = 0; j < U; j++) {
        const KvUnit u = kv_unit(tiles, from + j * 256 + threadIdx.x);
        places[j] = __shfl(rows.place, (int)u.row, 64);
        pages[j] = (uint32_t)__shfl((int)rows.page, (int)u.row, 64);
        if (u.row >= count || u.unit >= tiles.units) places[j] = -1;
        const uint32_t slot = u.unit >> words_log2, e0 = (u.unit & (words - 1u)) * 8;
        if (places[j] >= 0) in[j].load(a, base_of(slot), index_of(row0 + u.row, slot), e0, (uint32_t)places[j], slot < a.hq + kv.hkv);
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
        if (places[j] < 0) continue;   // (whole heads)
        const KvUnit u = kv_unit(tiles, from + j * 256 + threadIdx.x);
        const uint32_t slot = u.unit >> words_log2, e0 = (u.unit & (words - 1u)) * 8, place = (uint32_t)places[j], page = pages[j], head = head_of(slot);
        const uint64_t row = row0 + u.row;
        const bool value = slot >= a.hq + kv.hkv;
        float v[8];
        in[j].values(a, base_of(slot), index_of(row, slot), e0, place, !value, v);
        if (slot < a.hq) {
            kv_store8<DT, (U > 1)>(a.q_out, row * a.q_out_stride + (uint64_t)slot * kv.dim + e0, v);
            continue;
        }
        float mn = v[0], mx = v[0];
        bool fine = true;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            fine = fine && fabsf(v[i]) < INFINITY;
            mn = v[i] < mn ? v[i] : mn;
            mx = v[i] > mx ? v[i] : mx;
        }
        uint32_t all_fine = fine;
        for (uint32_t d = 1; d < kv.group / 8; d <<= 1) {   // (a group's lanes are neighbours and within a head)
            const float omn = __shfl_xor(mn, (int)d, 64), omx = __shfl_xor(mx, (int)d, 64);
            mn = omn < mn ? omn : mn;
            mx = omx > mx ? omx : mx;
            all_fine &= (uint32_t)__shfl_xor((int)all_fine, (int)d, 64);
        }
        float scale = (mx - mn) / 15.0f;
        if (scale < 1.0e-7f) scale = 1.0f;
        const float inv = 1.0f / scale;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float d = v[i] - mn;
            const float p = d * inv;
            float q = p + 0.5f;
            q = q < 0.0f ? 0.0f : q;
            q = q > 15.0f ? 15.0f : q;
            word |= (uint32_t)q << (4 * i);
        }
        if (!all_fine) {   // reads as NaN, all of it
            scale = mn = __builtin_nanf("");
            word = 0;
        }
        if (page >= kv.n_pages) continue;
        const uint64_t to = (((uint64_t)page * kv.hkv + head) << kv.page_log2) + (place & ((1u << kv.page_log2) - 1u));
        (value ? kv.v.codes : kv.k.codes)[to * words + e0 / 8] = word;
        if (e0 % kv.group == 0) {
            const uint64_t g = to * (kv.dim / kv.group) + e0 / kv.group;
            store_elem<DT>(value ? kv.v.scales : kv.k.scales, g, scale);
            store_elem<DT>(value ? kv.v.biases : kv.k.biases, g, mn);
        }
    }
}

// Units are words of codes: the key heads', then the value heads' (what is not wanted has none); `keys` of them are keys'.
template <int DT, int U> __global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a, KvTiles tiles, uint32_t keys) {
#pragma clang fp contract(off)
    const KvArgs& kv = a.kv;
    const uint32_t tile = blockIdx.x / tiles.parts, row0 = tile * tiles.per_tile, from = (blockIdx.x - tile * tiles.parts) * (256 * U);
    const uint32_t count = kv.n_tokens - row0 < tiles.per_tile ? kv.n_tokens - row0 : tiles.per_tile;
    const KvRow rows = kv_rows(kv, row0, count);
    const uint32_t words = kv.dim / 8, words_log2 = (uint32_t)__builtin_ctz(words), groups = kv.dim / kv.group;
    uint32_t word[U];
    float scale[U], bias[U];
    uint64_t to[U];
    void* out[U];
#pragma unroll
    for (int j = 0; j < U; j++) {
        const KvUnit u = kv_unit(tiles, from + j * 256 + threadIdx.x);
        const int32_t place = __shfl(rows.place, (int)u.row, 64);
        const uint32_t page = (uint32_t)__shfl((int)rows.page, (int)u.row, 64);
        out[j] = nullptr;
        if (u.row >= count || u.unit >= tiles.units || place < 0 || page >= kv.n_pages) continue;
        const bool value = u.unit >= keys;
        const uint32_t unit = value ? u.unit - keys : u.unit, head = unit >> words_log2, w = unit & (words - 1u);
        const uint64_t at = (((uint64_t)page * kv.hkv + head) << kv.page_log2) + ((uint32_t)place & ((1u << kv.page_log2) - 1u)), g = at * groups + w * 8 / kv.group;
        word[j] = (value ? kv.v.codes : kv.k.codes)[at * words + w];
        scale[j] = load_elem<DT>(value ? kv.v.scales : kv.k.scales, g);
        bias[j] = load_elem<DT>(value ? kv.v.biases : kv.k.biases, g);
        out[j] = value ? a.v : a.k;
        to[j] = ((uint64_t)(row0 + u.row) * kv.hkv + head) * kv.dim + 8 * w;
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
        if (!out[j]) continue;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float p = scale[j] * (float)(word[j] >> (4 * i) & 15u);
            v[i] = p + bias[j];
        }
        kv_store8<DT, (U > 1)>(out[j], to[j], v);
    }
}

// Tiles of rows for workgroups of 256 threads with `each` units a thread: whole rows while a workgroup has several, else parts of one.
bool tiles_of(uint32_t n_tokens, uint64_t units, uint32_t each, KvTiles& t, uint64_t& groups) {
    const uint32_t room = 256 * each;
    t.units = (uint32_t)units;
    t.per_tile = units < room ? (uint32_t)(room / units) : 1u;
    if (t.per_tile > 64) t.per_tile = 64;
    t.parts = (uint32_t)((units * t.per_tile + room - 1) / room);
    t.magic = t.units > 1 ? (uint32_t)(((1ull << 32) + units - 1) / units) : 0u;
    groups = (uint64_t)((n_tokens + t.per_tile - 1) / t.per_tile) * t.parts;
    return groups <= max_workgroups(256);
}
template <int U, int DT> const void* append_kernel_of(int pairs) {
    switch (pairs) {
        case KV_PLAIN: return (const void*)kv_append_kernel<DT, KV_PLAIN, U>;
        case KV_NEIGHBOURS: return (const void*)kv_append_kernel<DT, KV_NEIGHBOURS, U>;
        case KV_HALVES: return (const void*)kv_append_kernel<DT, KV_HALVES, U>;
        default: return (const void*)kv_append_kernel<DT, KV_ANY, U>;
    }
}
template <int U> const void* append_kernel(int dtype, int pairs) {
    return dtype == DT_F32 ? append_kernel_of<U, DT_F32>(pairs) : dtype == DT_F16 ? append_kernel_of<U, DT_F16>(pairs) : append_kernel_of<U, DT_BF16>(pairs);
}
// Several units a thread where that leaves the chip full: their loads are under way together.
uint32_t units_each(uint32_t n_tokens, uint64_t units, uint32_t most) { return (uint64_t)n_tokens * units >= 256ull * most * 512 ? most : 1u; }

}  // namespace

int launch_kv_append(int dtype, const KvAppendArgs& p, const LaunchCtx& lc) {
    KvAppendArgs a = p;
    const uint64_t units = (uint64_t)(a.hq + 2 * a.kv.hkv) * (a.kv.dim / 8);
    const uint32_t each = units_each(a.kv.n_tokens, units, 4);
    KvTiles t;
    uint64_t groups;
    if (!tiles_of(a.kv.n_tokens, units, each, t, groups)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    const int pairs = !a.rot ? KV_PLAIN : a.rot % (a.neighbours ? 8 : 16) ? KV_ANY : a.neighbours ? KV_NEIGHBOURS : KV_HALVES;
    const void* fn = each > 1 ? append_kernel<4>(dtype, pairs) : append_kernel<1>(dtype, pairs);
    void* args[] = {&a, &t};
    MTQ_HIP(launch_kernel(fn, dim3((uint32_t)groups), dim3(256), args, 0, lc));
    return ERR_OK;
}

int launch_kv_read(int dtype, const KvReadArgs& p, const LaunchCtx& lc) {
    KvReadArgs a = p;
    const uint64_t one = (uint64_t)a.kv.hkv * (a.kv.dim / 8), units = (a.k ? one : 0) + (a.v ? one : 0);
    uint32_t keys = a.k ? (uint32_t)one : 0;
    const uint32_t each = units_each(a.kv.n_tokens, units, 4);
    KvTiles t;
    uint64_t groups;
    if (!tiles_of(a.kv.n_tokens, units, each, t, groups)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    const void* fn[2][3] = {{(const void*)kv_read_kernel<DT_F32, 1>, (const void*)kv_read_kernel<DT_F16, 1>, (const void*)kv_read_kernel<DT_BF16, 1>},
                            {(const void*)kv_read_kernel<DT_F32, 4>, (const void*)kv_read_kernel<DT_F16, 4>, (const void*)kv_read_kernel<DT_BF16, 4>}};
    void* args[] = {&a, &t, &keys};
    MTQ_HIP(launch_kernel(fn[each > 1][dtype], dim3((uint32_t)groups), dim3(256), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
