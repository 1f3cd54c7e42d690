// Log probabilities of given tokens, entropy and top alternatives of rows of logits: what a server answers with, behind the
// output head.
//
//   m = max x,  z = sum exp(x - m),  s = sum exp(x - m) (x - m)
//   log p(t) = (x_t - m) - log z,    entropy = log z - s / z
//
// One read of the logits bounds it: everything else is a few numbers a row. Each lane runs through its part of a row with the
// maximum so far and both sums relative to it (a larger maximum d above the old one turns z into z e^-d and s into (s - d z) e^-d),
// so nothing is read twice and no exponent overflows. Sums, maxima and logarithms are f32 for every element type, and results are
// not rounded to it.
//
// The top k come from the same pass. A wave keeps a list of candidates in LDS, a 64-bit key each: the logit's bits in an order of
// unsigned integers, and below them the complement of the index, so that keys are distinct and equal logits go to the lower index.
// An element joins the list if its key is above a bar that at least k of the wave's elements have reached; a lane's vectors are
// asked for their maxima first, which the running maximum needs anyway, so that a wave pays for the list only where it grows
// (k ln(n / k) times over n elements in no order). A wave whose list is long draws its top k out of it, and the k-th becomes the bar.
#include "mtq_device.h"
#include "mtq_internal.h"

namespace mtq {

namespace {

constexpr uint32_t kTopMost = 32;        // alternatives a row
constexpr uint32_t kListCap = 576;       // a wave's candidates: 32 kept, and a vector of 8 elements of 64 lanes
constexpr uint32_t kTileElems = 32;      // elements of a lane's tile: 64 bytes of 16-bit logits, 128 of f32
constexpr int kWaves = 4;

struct LogprobArgs {
    const void* logits;
    uint64_t stride;            // elements between rows
    const uint32_t* tokens;     // [rows, n_given]
    float* token_logprobs;      // [rows, n_given]
    float* entropy;             // [rows]
    uint32_t* top_ids;          // [rows, k]
    float* top_logprobs;
    float* part;                // [rows, slices, 4]: m, z, s
    uint64_t* part_keys;        // [rows, slices, k]
    uint32_t n_given, k, vocab, slices;
};

__device__ __forceinline__ uint32_t ordered(float v) {   // unsigned order; -0 as 0
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// What a lane, and then a wave, has seen of a row.
struct Seen {
    float m = -INFINITY, z = 0.f, s = 0.f;
    // The sums relative to a maximum that is not below m.
    __device__ __forceinline__ void raise(float to) {
        if (to > m) {
            if (z != 0.f) {   // (nothing summed yet: no difference to take)
                const float d = m - to, f = __expf(d);
                s = f > 0.f ? (s + d * z) * f : 0.f;
                z *= f;
            }
            m = to;
        }
    }
    __device__ __forceinline__ void join(float m2, float z2, float s2) {
        Seen o;
        o.m = m2; o.z = z2; o.s = s2;
        const float top = fmaxf(m, o.m);
        raise(top);
        o.raise(top);
        z += o.z;
        s += o.s;
    }
    __device__ __forceinline__ void join_lanes() {
        float top = m;
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        raise(top);
        z = seg_allreduce(z, 64);
        s = seg_allreduce(s, 64);
    }
};

// The top `k` of the wave's `n` keys in list[0 .. n), in order, to out[0 .. k) (0: no more keys); returns the k-th. `spare` has room for k;
// out may be `list`. Keys other than 0 are distinct: a lane counts for each of its keys how many of all are larger (reads of LDS that all
// lanes share), and the count is the key's place.
template <int P> __device__ __forceinline__ void place_top(const uint64_t* list, uint32_t from, uint32_t n, uint64_t* out, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    uint64_t mine[P];
    uint32_t above[P] = {};
#pragma unroll
    for (int i = 0; i < P; i++) mine[i] = from + i * 64 + lane < n ? list[from + i * 64 + lane] : 0;
    uint32_t j = 0;
    for (; j + 4 <= n; j += 4) {
        uint64_t o[4];
#pragma unroll
        for (int u = 0; u < 4; u++) o[u] = list[j + u];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < P; i++) above[i] += o[u] > mine[i];
    }
    for (; j < n; j++) {
        const uint64_t o = list[j];
#pragma unroll
        for (int i = 0; i < P; i++) above[i] += o > mine[i];
    }
#pragma unroll
    for (int i = 0; i < P; i++)
        if (mine[i] && above[i] < k) out[above[i]] = mine[i];
}
__device__ __forceinline__ uint64_t draw_top(const uint64_t* list, uint32_t n, uint64_t* spare, uint64_t* out, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    auto turned = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };   // (LDS operations of a wave complete in order)
    turned();
    if (lane < k) spare[lane] = 0;
    turned();
    if (n <= 64) place_top<1>(list, 0, n, spare, k);
    else
        for (uint32_t from = 0; from < n; from += 128) place_top<2>(list, from, n, spare, k);
    turned();
    const uint64_t mine = lane < k ? spare[lane] : 0, last = spare[k - 1];
    if (lane < k) out[lane] = mine;
    turned();
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(last >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)last);
}

// A row's given tokens' logits, the first 64 of them: asked for before anything else of the row.
template <int DT> struct Given {
    uint32_t id = 0xFFFFFFFFu;
    float x = 0.f;
    __device__ __forceinline__ void load(const LogprobArgs& a, uint32_t row, uint32_t j) {
        id = j < a.n_given ? a.tokens[(uint64_t)row * a.n_given + j] : 0xFFFFFFFFu;
        if (id < a.vocab) x = load_elem<DT>(a.logits, (size_t)row * a.stride + id);
    }
};

// A row's results, by one wave: z and s relative to m, keys in order.
template <int DT> __device__ __forceinline__ void finish(const LogprobArgs& a, uint32_t row, const Seen& t, const uint64_t* keys, Given<DT> given) {
    const uint32_t lane = threadIdx.x & 63u;
    // No token has any probability where every logit is -inf (z = 0): log probabilities are -inf, the entropy 0. A NaN or +inf among
    // the logits makes z NaN, and all of the row's results with it.
    const bool none = t.z == 0.f;
    const float log_z = none ? 0.f : logf(t.z);
    auto lp = [&](float x) { return none ? -INFINITY : (x - t.m) - log_z; };
    if (a.entropy && lane == 0) a.entropy[row] = none ? 0.f : log_z - t.s / t.z;
    for (uint32_t j = lane; j < a.n_given; j += 64) {
        if (j >= 64) given.load(a, row, j);
        if (given.id < a.vocab) a.token_logprobs[(uint64_t)row * a.n_given + j] = lp(given.x);
    }
    if (lane < a.k) {
        const uint64_t key = keys[lane], at = (uint64_t)row * a.k + lane;
        if (a.top_ids) a.top_ids[at] = ~(uint32_t)key;             // (0, no key: 0xFFFFFFFF)
        if (a.top_logprobs) a.top_logprobs[at] = key ? lp(unordered((uint32_t)(key >> 32))) : NAN;
    }
}

struct WaveLists {
    uint64_t list[kWaves][kListCap], spare[kWaves][kTopMost], comb[kWaves * kTopMost];
    float sums[kWaves][3];
};

// A wave's candidates.
struct Candidates {
    uint64_t *list, *spare;
    uint32_t n = 0, k;
    uint64_t bar = 0;            // keys above it join
    float bar_value = -INFINITY; // no smaller logit has such a key
    __device__ __forceinline__ void draw() {
        const uint64_t kth = draw_top(list, n, spare, list, k);
        n = n < k ? n : k;
        if (kth) raise_bar(kth);
    }
    __device__ __forceinline__ void raise_bar(uint64_t key) {
        bar = key;
        bar_value = unordered((uint32_t)(key >> 32));
    }
};

// What the workgroup's waves have seen and the top k of their lists, joined in its first wave (all of its lanes get it); keys to `comb`.
__device__ __forceinline__ Seen join_waves(Seen t, const Candidates& c, WaveLists& w) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    t.join_lanes();
    if (c.k) draw_top(c.list, c.n, c.spare, w.comb + wave * c.k, c.k);
    if (lane == 0) { w.sums[wave][0] = t.m; w.sums[wave][1] = t.z; w.sums[wave][2] = t.s; }
    __syncthreads();
    if (wave == 0) {
        Seen all;
        if (lane < kWaves) { all.m = w.sums[lane][0]; all.z = w.sums[lane][1]; all.s = w.sums[lane][2]; }
        all.join_lanes();
        t = all;
        if (c.k) draw_top(w.comb, kWaves * c.k, c.spare, w.comb, c.k);
    }
    return t;
}

// Workgroup (slice, row): its four waves take tiles of 64 lanes x 32 elements in turn, the next tile's on its way while one is worked on. The
// row's vectors are the 16-byte blocks of memory that hold any of it, so that rows of every alignment are read in whole vectors; elements
// before and behind the row count as nothing.
template <int DT> __global__ __launch_bounds__(64 * kWaves, 4) void logprobs_kernel(LogprobArgs a) {
    constexpr int ES = DT == DT_F32 ? 4 : 2, PER = 16 / ES, NV = kTileElems / PER;
    __shared__ WaveLists lds;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const uint64_t at = (uint64_t)(uintptr_t)a.logits + (uint64_t)row * a.stride * ES;
    const uint32_t skip = (uint32_t)(at & 15u) / ES;                          // elements of the first vector that are not the row's
    const uint4* vecs = (const uint4*)(at & ~(uint64_t)15);
    const uint32_t n_vecs = (skip + a.vocab + PER - 1) / PER;
    constexpr uint32_t kTileVecs = 64 * NV;
    const uint32_t n_tiles = (n_vecs + kTileVecs - 1) / kTileVecs;
    Candidates c;
    c.list = lds.list[wave];
    c.spare = lds.spare[wave];
    c.k = a.k;
    bool open = true;                // no bar yet
    Seen t;
    uint4 raw[NV], next[NV];
    auto load = [&](uint32_t tile) {
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const uint32_t v = tile * kTileVecs + lane + u * 64;
            next[u] = v < n_vecs ? vecs[v] : make_uint4(0, 0, 0, 0);
        }
    };
    auto value = [](const uint4& r, int j) -> float {
        const uint32_t w = ((const uint32_t*)&r)[ES == 4 ? j : j >> 1];
        if constexpr (DT == DT_F32) return __uint_as_float(w);
        else if constexpr (DT == DT_BF16) return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
        else return f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu);
    };
    load(slice * kWaves + wave);
    Given<DT> given;
    if (a.slices == 1 && wave == 0) given.load(a, row, lane);
    for (uint32_t tile = slice * kWaves + wave; tile < n_tiles; tile += a.slices * kWaves) {
#pragma unroll
        for (int u = 0; u < NV; u++) raw[u] = next[u];
        load(tile + a.slices * kWaves);
        const uint32_t v0 = tile * kTileVecs + lane;
        const bool edge = tile == 0 || tile == n_tiles - 1;
        float vmax[NV], x[NV][PER];
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < NV; u++) {
            vmax[u] = -INFINITY;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                x[u][j] = value(raw[u], j);
                if (edge) {
                    const uint32_t e = (v0 + u * 64) * PER + j - skip;        // (before the row: wraps past vocab)
                    if (e >= a.vocab) x[u][j] = -INFINITY;
                }
                vmax[u] = fmaxf(vmax[u], x[u][j]);
            }
            top = fmaxf(top, vmax[u]);
        }
        t.raise(top);
        const float base = t.m == -INFINITY ? 0.f : t.m;
        float z = 0.f, s = 0.f;
#pragma unroll
        for (int u = 0; u < NV; u++)
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const float d = x[u][j] - base, e = __expf(d);
                z += e;
                s += e * fmaxf(d, -200.f);                                    // (e^-200 is 0, and 0 * -200 no NaN)
            }
        t.z += z;
        t.s += s;
        if (!c.k) continue;
        if (open) {
            // A first bar: the k-th largest of the lanes' maxima, bit by bit, is reached by k elements, and by few more. (What 16-bit types leave
            // below their bits is the same for all values of a sign.)
            constexpr int LOW = DT == DT_F32 ? 0 : DT == DT_F16 ? 13 : 16;
            const uint32_t o = ordered(top);
            uint32_t kth = 0;
#pragma unroll
            for (int b = 31; b >= LOW; b--) {
                const uint32_t to = kth | 1u << b;
                kth = (uint32_t)__popcll(__ballot(o >= to)) >= c.k ? to : kth;
            }
            c.raise_bar(((uint64_t)kth << 32) - 1);
            c.bar_value = unordered(kth);
        }
        const bool more = tile + a.slices * kWaves < n_tiles;
        if (__ballot(!(top < c.bar_value))) {
            uint32_t hot = 0;
#pragma unroll
            for (int u = 0; u < NV; u++) hot |= __ballot(!(vmax[u] < c.bar_value)) ? 1u << u : 0u;
            while (hot) {
                const uint32_t u = __builtin_ctz(hot);
                hot &= hot - 1;
                uint4 r = raw[0];
#pragma unroll
                for (int i = 1; i < NV; i++)
                    if (u == i) r = raw[i];
                if (c.n + 64 * PER > kListCap) {                              // (a vector of candidates might not fit)
                    uint32_t most = 0;
#pragma unroll
                    for (int j = 0; j < PER; j++) most += __popcll(__ballot(!(value(r, j) < c.bar_value)));
                    if (c.n + most > kListCap) c.draw();                      // (then they fit: at most 32 and 512)
                }
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const float v = value(r, j);
                    if (!__ballot(!(v < c.bar_value))) continue;
                    const uint32_t e = (v0 + u * 64) * PER + j - skip;
                    const uint64_t key = v == v && e < a.vocab ? (uint64_t)ordered(v) << 32 | (uint32_t)~e : 0;
                    const uint64_t who = __ballot(key > c.bar);
                    if (key > c.bar) c.list[c.n + __popcll(who & ((1ull << lane) - 1))] = key;
                    c.n += __popcll(who);
                }
            }
            if (more && c.n > c.k + 12) c.draw();
        }
        open = false;
    }
    t = join_waves(t, c, lds);
    if (wave) return;
    if (a.slices == 1) {
        finish<DT>(a, row, t, lds.comb, given);
    } else {
        const size_t i = (size_t)row * a.slices + slice;
        if (lane == 0) { a.part[4 * i] = t.m; a.part[4 * i + 1] = t.z; a.part[4 * i + 2] = t.s; }
        if (lane < a.k) a.part_keys[i * a.k + lane] = lds.comb[lane];
    }
}

// A row's slices joined by one workgroup: at most kSlicesMost, so that their keys fit the waves' lists. (A launch of its own: the last slice's
// workgroup joining them behind a fence took longer, 33 x 50257 f32 with 20 alternatives 24.5 us against 17.9.)
constexpr uint32_t kSlicesMost = 32;
static_assert(kSlicesMost / kWaves * kTopMost <= kListCap && kSlicesMost <= 64, "a wave's share of the slices fits its list and its lanes");
template <int DT> __global__ __launch_bounds__(64 * kWaves) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ WaveLists lds;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
    Given<DT> given;
    if (wave == 0) given.load(a, row, lane);
    const uint32_t mine = (a.slices + kWaves - 1) / kWaves, from = wave * mine < a.slices ? wave * mine : a.slices;
    const uint32_t to = from + mine < a.slices ? from + mine : a.slices;
    Candidates c;
    c.list = lds.list[wave];
    c.spare = lds.spare[wave];
    c.k = a.k;
    c.n = (to - from) * a.k;
    const uint64_t* keys = a.part_keys + ((size_t)row * a.slices + from) * a.k;
    for (uint32_t i = lane; i < c.n; i += 64) c.list[i] = keys[i];
    Seen t;
    if (from + lane < to) {
        const float* p = a.part + 4 * ((size_t)row * a.slices + from + lane);
        t.m = p[0]; t.z = p[1]; t.s = p[2];
    }
    t = join_waves(t, c, lds);
    if (wave == 0) finish<DT>(a, row, t, lds.comb, given);
}

}  // namespace

static uint32_t logprob_slices(uint32_t rows, uint32_t vocab) {
    const uint32_t tiles = vocab / (64 * kTileElems) + 1, most = (tiles + kWaves - 1) / kWaves;
    uint32_t s = rows >= 1024 ? 1 : 1024 / rows;
    if (s > most) s = most;
    return s > kSlicesMost ? kSlicesMost : s;
}

size_t logprobs_scratch_bytes(uint32_t rows, uint32_t vocab, uint32_t k) {
    const uint32_t s = logprob_slices(rows, vocab);
    return s == 1 ? 0 : (size_t)rows * s * (16 + 8 * k);
}

int launch_logprobs(int dtype, const void* logits, size_t stride, const uint32_t* tokens, uint32_t n_given, float* token_logprobs, float* entropy,
                    uint32_t* top_ids, float* top_logprobs, uint32_t k, uint32_t rows, uint32_t vocab, void* scratch, const LaunchCtx& lc) {
    LogprobArgs a;
    a.logits = logits; a.stride = stride; a.tokens = tokens; a.token_logprobs = token_logprobs; a.entropy = entropy; a.top_ids = top_ids;
    a.top_logprobs = top_logprobs; a.n_given = n_given; a.k = k; a.vocab = vocab;
    a.slices = scratch ? logprob_slices(rows, vocab) : 1;
    a.part = (float*)scratch;
    a.part_keys = scratch ? (uint64_t*)((char*)scratch + (size_t)rows * a.slices * 16) : nullptr;
    if ((uint64_t)rows * a.slices > max_workgroups(64 * kWaves)) return fail(ERR_SHAPE, "more rows than a launch can have workgroups");
    const void* fn = dtype == DT_F32 ? (const void*)logprobs_kernel<DT_F32> : dtype == DT_F16 ? (const void*)logprobs_kernel<DT_F16> : (const void*)logprobs_kernel<DT_BF16>;
    void* args[] = {&a};
    LaunchCtx first = lc;
    if (a.slices > 1) first.stop = nullptr;
    MTQ_HIP(launch_kernel(fn, dim3(rows * a.slices), dim3(64 * kWaves), args, 0, first));
    if (a.slices == 1) return ERR_OK;
    fn = dtype == DT_F32 ? (const void*)logprobs_join_kernel<DT_F32> : dtype == DT_F16 ? (const void*)logprobs_join_kernel<DT_F16> : (const void*)logprobs_join_kernel<DT_BF16>;
    LaunchCtx last = lc;
    last.start = nullptr;
    MTQ_HIP(launch_kernel(fn, dim3(rows), dim3(64 * kWaves), args, 0, last));
    return ERR_OK;
}

}  // namespace mtq
