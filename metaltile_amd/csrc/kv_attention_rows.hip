// Attention over the 4-bit cache for sequences of few rows (single tokens, drafts).
//
// A workgroup has 16 rows (of a sequence's new tokens times the query heads that share a key head) and a piece of its tokens, each of its four waves a run of that, 32 tokens
// at a time, which come into its own part of the LDS by load-to-LDS instructions a block ahead: no register holds what is on its way, and no wave waits for another until
// all have their sums. 16 tokens lie on one page. Pieces of 16 bytes go into the LDS by piece and token, so that the words that a matrix instruction takes at once
// lie in different banks. The values' words have eight numbers of one token, while the instruction wants numbers of eight tokens: byte by byte two tokens'
// words are put together, each lane with its number's nibble turned to the place first (kv_attention.h has the arithmetic).
// Bound by the vector units from 16 rows on, which have 419 instructions for 32 tokens, and by latency in small calls: 32 sequences of 4096 tokens, 16 rows, bf16: 48 us
// (3.2 TB/s); one of 1000 tokens 11 us, of which the join is 4; 12 sequences of up to 1024 visible tokens, 10 rows, f32: 15 us.
#include "kv_attention.h"

namespace mtq {

namespace {

// Sizes of a wave's part of the LDS, in bytes.
template <int DT, int D, int G> struct RowsLds {
    static constexpr int ES = DT == DT_F32 ? 4 : 2, NG = D / G;
    static constexpr int CODES = 16 * D;                         // of 32 tokens' keys, or values
    static constexpr int HALF = 16 * NG * ES;                    // of 16 tokens' scales, or biases
    static constexpr int LOADS = HALF * 4 > 256 ? HALF * 4 / 256 : 1;   // that bring scales and biases of 32 tokens, of keys or values
    static constexpr int STAGE = 2 * CODES + 2 * LOADS * 256;
    static constexpr int JOIN = 16 * (D + 4) * 4;                // rows' values, and behind each its maximum and sum
    static constexpr int WAVE = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
    static constexpr int NW = 4;   // waves
    // Of a SIMD at a time, by the registers: with more of them an instance spills (256 values in groups of 32, f32: 370 us with one wave, 987 with two; bf16 225 / 337).
    static constexpr int AT_ONCE = DT != DT_F32 && D <= 128 && G >= 64 ? 3 : D == 256 && (DT == DT_F32 || G == 32 || (DT == DT_F16 && G == 64)) ? 1 : 2;
    static_assert(NW * WAVE <= 160 * 1024, "");
};

// The values' number (row of the matrix instruction) `m` of tile t of a group, as its place in the group.
template <int G> __device__ __forceinline__ uint32_t kv_number(uint32_t t, uint32_t m) {
    constexpr uint32_t W = G / 8;   // words of a group
    return 8 * (m % W) + (16 / W) * t + m / W;
}

template <int DT, int D, int G>
__global__ __launch_bounds__(256, (RowsLds<DT, D, G>::AT_ONCE)) void kv_rows_kernel(KvAttentionArgs a, KvParts parts) {
    using L = RowsLds<DT, D, G>;
    using T = KvTerms<DT>;
    constexpr int NW = L::NW, STEPS = D / 32, NG = D / G, NT = G / 16, ES = L::ES, W = G / 8;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15u, g = lane >> 4;
    const uint32_t head = blockIdx.x % kv.hkv, shared = a.hq / kv.hkv;
    KvPiece piece;
    if (!kv_piece<16>(a, parts, blockIdx.x / kv.hkv, piece)) return;   // (all of the workgroup's waves find the same)
    const KvSeq& s = piece.s;
    const uint32_t slice = piece.slice, slices = piece.slices;
    uint8_t* mine = lds + wave * L::WAVE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
    const uint32_t rows = s.rows * shared;   // (fewer than 2^24 2^16: checked against the launch on the host)
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);   // (not 0: what is hidden scores -inf)
    const uint32_t k16 = kv_sixteen<T::QK>(), v16 = kv_sixteen<DT_BF16>();

    const uint32_t row0 = piece.set * 16;
    // This lane's row sees tokens from .. end - 1.
    const uint32_t index = row0 + r, last = row0 + 15u < rows ? row0 + 15u : rows - 1u;
    auto end_of = [&](uint32_t i) { const int32_t e = (int32_t)(s.len + i / shared + 1u) - (int32_t)s.rows; return e > 0 ? (uint32_t)e : 0u; };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    const bool alive = index < rows;
    const uint32_t token = (alive ? index : last) / shared, qh = head * shared + (alive ? index : last) % shared, end = end_of(alive ? index : last), from = from_of(end);
    const uint32_t first_end = __builtin_amdgcn_readfirstlane(end_of(row0)), last_end = __builtin_amdgcn_readfirstlane(end_of(last));
    const uint32_t lo = from_of(first_end) & ~31u, last_from = from_of(last_end);
    const uint32_t blocks = kv.n_pages && last_end > lo ? (last_end - lo + 31u) / 32u : 0u;
    const uint32_t workers = slices * NW, per = (blocks + workers - 1u) / workers;
    const uint32_t b0 = (slice * NW + wave) * per < blocks ? (slice * NW + wave) * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;

    // Queries: words 4 i + g of the codes' rows meet values 32 i + 8 g .. + 7, in the order in which a word's nibbles come out.
    kr_u32x4 q[T::Q][STEPS];
    float qsum[NG] = {};
    const uint64_t q_at = (uint64_t)(s.first_row + token) * a.q_stride + (uint64_t)qh * D + 8 * g;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = load_elem<DT>(a.q, q_at + 32 * i + j);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = a.scale < 0.f ? -v[j] : v[j];
            qsum[i * 32 / G] += v[j];
        }
#pragma unroll
        for (int p = 0; p < 4; p++) {
            if constexpr (DT == DT_F16) {
                q[0][i][p] = (uint32_t)f32_to_elem_bits<DT_F16>(v[p]) | (uint32_t)f32_to_elem_bits<DT_F16>(v[p + 4]) << 16;
            } else {
                float x[T::Q], y[T::Q];
                kv_split(v[p], x);
                kv_split(v[p + 4], y);
#pragma unroll
                for (int t = 0; t < T::Q; t++) q[t][i][p] = kv_pack_bf16(x[t], y[t]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NG; n++) qsum[n] = kv_column_sum(qsum[n]);

    // Pages of 64 sixteens of tokens at a time, one to a lane.
    uint32_t page = 0, page_from = 0xFFFFFFFFu;
    auto pages_at = [&](uint32_t h) {
        page_from = h;
        const uint32_t at = (h + lane) * 16u;
        page = at < last_end ? kv.pages[(uint64_t)s.seq * kv.pages_stride + (at >> kv.page_log2)] : 0xFFFFFFFFu;
    };
    auto half_of = [&](uint32_t h) { return __builtin_amdgcn_readlane(page, h - page_from); };   // sixteen h's page
    auto slot_of = [&](uint32_t pg, uint32_t h) {   // its index [page, head, place] (of no page: one that is there)
        const uint32_t p = pg < kv.n_pages ? pg : 0u;
        return ((((uint64_t)p * kv.hkv + head) << kv.page_log2) + ((h * 16u) & ((1u << kv.page_log2) - 1u)));
    };
    auto issue = [&](uint32_t b) {   // block b's loads, 2 (D / 64 + LOADS) of them
        const uint32_t h = lo / 16u + 2u * b, to = lds0 + (b & 1u) * L::STAGE;
        const uint64_t sa = slot_of(half_of(h), h), sb = slot_of(half_of(h + 1u), h + 1u);
#pragma unroll
        for (int part = 0; part < 2; part++) {
            const KvPart& x = part ? kv.v : kv.k;
            const uint32_t at = to + part * (L::CODES + L::LOADS * 256);
#pragma unroll
            for (int u = 0; u < D / 64; u++) {   // piece and token of 16 bytes: piece p of token t of a half at p * 16 + t
                const uint32_t p = u * 64 + lane, half = p / (D / 2), piece = p % (D / 2) / 16, t = p % 16;
                kv_load16(__builtin_amdgcn_readfirstlane(at + u * 1024), (const uint8_t*)x.codes + ((half ? sb : sa) + t) * (D / 2) + piece * 16);
            }
#pragma unroll
            for (int u = 0; u < L::LOADS; u++) {   // scales of both halves, then biases
                const uint32_t p = (u * 256 + lane * 4) % (L::HALF * 4), half = p / L::HALF % 2;
                const uint8_t* base = p >= 2 * L::HALF ? (const uint8_t*)x.biases : (const uint8_t*)x.scales;
                kv_load4(__builtin_amdgcn_readfirstlane(at + L::CODES + u * 256), base + (half ? sb : sa) * (NG * ES) + p % L::HALF);
            }
        }
    };

    kr_f32x4 o[NG][NT] = {};   // values by group and tile
    float ones[NG] = {}, bias[NG] = {}, sum = 0.f, bar = -INFINITY;   // (ones: -24 sum p s)
    auto block = [&](uint32_t b, bool whole) {   // whole: every row sees all of the block
        const uint8_t* at = mine + (b & 1u) * L::STAGE;
        const uint32_t t0 = lo + 32u * b, h = lo / 16u + 2u * b;
        // Scales or biases of this lane's tokens 4 g .. 4 g + 3 of a half, as they are stored, and one of them.
        struct Numbers {
            uint32_t w[NG * ES];
            __device__ __forceinline__ float operator()(int i, int n) const {
                const int e = i * NG + n;
                if constexpr (DT == DT_F32) return __uint_as_float(w[e]);
                else return kr_elem<DT>(w[e / 2], e & 1);
            }
            __device__ __forceinline__ void keep(int i, uint32_t yes) {   // or 0 in the place of token i's
                const uint32_t all = 0u - yes;
                if constexpr (NG * ES == 2) {
                    w[i / 2] &= i & 1 ? all | 0xFFFFu : all | 0xFFFF0000u;
                } else {
#pragma unroll
                    for (int j = 0; j < NG * ES / 4; j++) w[i * (NG * ES / 4) + j] &= all;
                }
            }
        };
        auto numbers = [&](const uint8_t* p, int array, int half) {
            Numbers v;
            const uint8_t* from8 = p + (array * 2 + half) * L::HALF + g * (4 * NG * ES);
#pragma unroll
            for (int i = 0; i < NG * ES; i += 2) {
                const uint2 two = *(const uint2*)(from8 + 4 * i);
                v.w[i] = two.x;
                v.w[i + 1] = two.y;
            }
            return v;
        };
        float x[2][4];   // scores, then weights
        uint32_t seen = 0xFFu;   // (a bit for each score: what is not whole is a small part of the blocks)
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            kr_f32x4 acc[NG];
#pragma unroll
            for (int n = 0; n < NG; n++) {
                const float start = T::CENTRED ? 0.f : -16.f * qsum[n];
                acc[n] = kr_f32x4{start, start, start, start};
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                const uint32_t w = *(const uint32_t*)(at + t * (L::CODES / 2) + i * 256 + (r * 4 + g) * 4);
                kr_u32x4 k;
#pragma unroll
                for (int p = 0; p < 4; p++) k[p] = kv_operand<DT>(kv_pair<T::QK>(w, p, k16));
#pragma unroll
                for (int e = T::Q - 1; e >= 0; e--) acc[i * 32 / G] = kr_mfma<T::QK>(k, q[e][i], acc[i * 32 / G]);
            }
            const Numbers ks = numbers(at + L::CODES, 0, t), kb = numbers(at + L::CODES, 1, t);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                auto rest = [&](int n) { return T::CENTRED ? fmaf(8.f, ks(i, n), kb(i, n)) : kb(i, n); };
                float v = ks(i, 0) * acc[0][i];
                v = fmaf(rest(0), qsum[0], v);
#pragma unroll
                for (int n = 1; n < NG; n++) v = fmaf(rest(n), qsum[n], fmaf(ks(i, n), acc[n][i], v));
                x[t][i] = v;
            }
            if (!whole) {
                const bool there = half_of(h + t) < kv.n_pages;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t tok = t0 + 16 * t + 4 * g + i;
                    if (!(there && tok >= from && tok < end)) {
                        x[t][i] = -INFINITY;
                        seen &= ~(1u << (4 * t + i));
                    }
                }
            }
            top = fmaxf(top, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            __builtin_amdgcn_sched_barrier(0);   // (one tile's operands at a time: what is asked for early has to be held)
        }
        if (__any(top * c > bar + kSlack)) {   // (base 2; of nothing seen: not so)
            const float to = fmaxf(bar, kv_column_max(top) * c);
            const float keep = to > bar ? __builtin_amdgcn_exp2f(bar - to) : 1.f;
            sum *= keep;
#pragma unroll
            for (int n = 0; n < NG; n++) {
                bias[n] *= keep;
                ones[n] *= keep;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][t][i] *= keep;
            }
            bar = to;
        }
        const float from_bar = bar == -INFINITY ? 0.f : bar;
        const uint8_t* values = at + L::CODES + L::LOADS * 256;
        Numbers vs[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            vs[t] = numbers(values + L::CODES, 0, t);
            Numbers vb = numbers(values + L::CODES, 1, t);
            if (!whole) {   // (a weight of 0 does not keep a NaN out)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    vs[t].keep(i, seen >> (4 * t + i) & 1u);
                    vb.keep(i, seen >> (4 * t + i) & 1u);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(x[t][i], c, -from_bar));
                x[t][i] = p;
                sum += p;
#pragma unroll
                for (int n = 0; n < NG; n++) bias[n] = fmaf(p, fmaf(8.f, vs[t](i, n), vb(i, n)), bias[n]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        const kr_u32x4 less24 = {0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u};   // -24 in bf16
#pragma unroll
        for (int n = 0; n < NG; n++) {
            kr_u32x4 pt[T::P];
#pragma unroll
            for (int j = 0; j < 4; j++) {   // tokens 4 g + 2 j, + 1 of the first half, then of the second
                float y[2][T::P];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = 2 * j % 4 + e;
                    kv_split(x[j / 2][i] * vs[j / 2](i, n), y[e]);
                }
#pragma unroll
                for (int e = 0; e < T::P; e++) pt[e][j] = kv_pack_bf16(y[0][e], y[1][e]);
            }
            kr_f32x4 less = {0.f, 0.f, 0.f, 0.f};   // (every row of it is the same)
            if constexpr (!T::CENTRED) {
#pragma unroll
                for (int e = T::P - 1; e >= 0; e--) less = kr_mfma<DT_BF16>(less24, pt[e], less);
            }
            const uint32_t word = n * W + r % W, sub = r / W;   // this lane's word of a token, and which of its nibbles
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = *(const uint32_t*)(values + j / 4 * (L::CODES / 2) + ((word / 4) * 16 + 4 * g + j % 4) * 16 + (word % 4) * 4);
            // W 16 (G 128): nibble t; W 8: nibble 2 t + sub, turned to bits 3..6 of byte t; W 4: nibble 4 t + sub, to bits 3..6 of half t.
            if constexpr (W != 16) {
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] = __builtin_amdgcn_alignbit(w[j], w[j], (4 * sub + 29) & 31);
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                kr_u32x4 v;
                const int byte = W == 16 ? t / 2 : W == 8 ? t : 2 * t;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t two = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x0C000C00u | (uint32_t)(4 + byte) << 16 | (uint32_t)byte);
                    if constexpr (W == 16) two = t & 1 ? two >> 1 : two << 3;
                    v[j] = kv_operand<DT>((two & 0x00780078u) | v16);
                }
#pragma unroll
                for (int e = T::P - 1; e >= 0; e--) o[n][t] = kr_mfma<DT_BF16>(v, pt[e], o[n][t]);
            }
            ones[n] += less[0];
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    constexpr int ON_WAY = 2 * (D / 64 + L::LOADS);
    if (b0 < b1) {
        auto refill = [&](uint32_t b) {   // the pages of block b and those behind it
            const uint32_t h = lo / 16u + 2u * b;
            if (page_from == 0xFFFFFFFFu || h + 1u - page_from > 63u) pages_at(h);
        };
        refill(b0);
        issue(b0);
        if (b0 + 1u < b1) issue(b0 + 1u);   // (pages of 32 blocks are there)
        for (uint32_t b = b0; b < b1; b++) {
            if (b + 1u < b1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ON_WAY) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const uint32_t t0 = lo + 32u * b, h = lo / 16u + 2u * b;
            const bool whole = t0 >= last_from && t0 + 32u <= first_end && half_of(h) < kv.n_pages && half_of(h + 1u) < kv.n_pages;
            block(b, whole);
            if (b + 2u < b1) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the stage is read)
                if (lo / 16u + 2u * (b + 2u) + 1u - page_from > 63u) pages_at(lo / 16u + 2u * (b + 1u));   // (the next block's are still asked for)
                issue(b + 2u);
            }
        }
    }

    // The waves' sums, relative to their bars, into the LDS; then joined.
    sum = kv_column_sum(sum);
    float* join = (float*)mine + r * (D + 4);
#pragma unroll
    for (int n = 0; n < NG; n++) {
        const float more = kv_column_sum(bias[n]) + ones[n];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) join[n * G + kv_number<G>(t, 4 * g + i)] = o[n][t][i] + more;
    }
    if (g == 0) {
        join[D] = bar;
        join[D + 1] = sum;
    }
    __syncthreads();
    const uint32_t count = rows - row0 < 16u ? rows - row0 : 16u;
    for (uint32_t u = threadIdx.x; u < count * (D / 4); u += 64 * NW) {
        const uint32_t row = u / (D / 4), d = u % (D / 4) * 4, i = row0 + row, tok = s.first_row + i / shared, h = head * shared + i % shared;
        const float* all = (const float*)lds + row * (D + 4);
        float top = -INFINITY, total = 0.f;
        for (int w = 0; w < NW; w++) top = fmaxf(top, all[w * (L::WAVE / 4) + D]);
        kr_f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < NW; w++) {
            const float* one = all + w * (L::WAVE / 4);
            const float part = one[D + 1], f = one[D] == -INFINITY ? (part == 0.f ? 0.f : 1.f) : exp2f(one[D] - top);   // (no bar and a sum: NaN)
            total = fmaf(part, f, total);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = f == 0.f && part == 0.f ? v[j] : fmaf(one[d + j], f, v[j]);
        }
        if (slices == 1) {
            const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int j = 0; j < 4; j++) store_elem<DT>(a.out, (uint64_t)tok * a.out_stride + (uint64_t)h * D + d + j, total == 0.f ? 0.f : v[j] * inv);
        } else {
            const uint64_t at = ((uint64_t)tok * a.hq + h) * parts.slices + slice;
            *(kr_f32x4*)(parts.values + at * D + d) = v;
            if (d == 0) {
                parts.sums[at * 2] = top;
                parts.sums[at * 2 + 1] = total;
            }
        }
        if (d == 0 && slice + 1u == slices && parts.slices > 1) {   // (of one slice: nothing to join)
            const uint32_t n = slices == 1 ? 0u : slices;
            if (n < parts.slices) parts.sums[(((uint64_t)tok * a.hq + h) * parts.slices + n) * 2 + 1] = kNoMore;
        }
    }
}

template <int DT, int D, int G> int launch(const KvAttentionArgs& p, KvParts parts, const LaunchCtx& lc) {
    using L = RowsLds<DT, D, G>;
    KvAttentionArgs a = p;
    const void* fn = (const void*)kv_rows_kernel<DT, D, G>;
    const size_t bytes = L::NW * L::WAVE;
    const uint64_t groups = kv_pieces<16>(a, parts);
    if (groups * a.kv.hkv > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    LaunchCtx first = lc, last = lc;
    if (parts.slices > 1) {
        first.stop = nullptr;
        last.start = nullptr;
    }
    MTQ_HIP(set_max_dynamic_lds(fn, bytes));
    void* args[] = {&a, &parts};
    MTQ_HIP(launch_kernel(fn, dim3((uint32_t)(groups * a.kv.hkv)), dim3(64 * L::NW), args, bytes, first));
    return parts.slices > 1 ? launch_kv_join(DT, a, parts, last) : ERR_OK;
}

template <int DT> int launch_of(const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (p.kv.dim * 1000 + p.kv.group) {
        case 64032: return launch<DT, 64, 32>(p, parts, lc);
        case 64064: return launch<DT, 64, 64>(p, parts, lc);
        case 128032: return launch<DT, 128, 32>(p, parts, lc);
        case 128064: return launch<DT, 128, 64>(p, parts, lc);
        case 128128: return launch<DT, 128, 128>(p, parts, lc);
        case 256032: return launch<DT, 256, 32>(p, parts, lc);
        case 256064: return launch<DT, 256, 64>(p, parts, lc);
        case 256128: return launch<DT, 256, 128>(p, parts, lc);
    }
    return fail(ERR_UNSUPPORTED, "kv_attention: no kernel for this head_dim and group_size");
}

}  // namespace

int launch_kv_rows(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (dtype) {
        case DT_F32: return launch_of<DT_F32>(p, parts, lc);
        case DT_F16: return launch_of<DT_F16>(p, parts, lc);
        default: return launch_of<DT_BF16>(p, parts, lc);
    }
}

}  // namespace mtq
