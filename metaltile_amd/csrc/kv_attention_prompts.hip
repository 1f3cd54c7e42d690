// Attention over the 4-bit cache for sequences of many rows (prompts), f16 and bf16: bound by the matrix cores.
//
// Keys and values are made s c + b in T first, once for all query heads and tiles, by a launch of its own (14 us for 8192 tokens of 8 heads of 128 values), in
// the order in which the instructions take them. With the codes themselves as operands (kv_attention_tiles.hip) every score and weight is scaled by its group in f32, and every
// tile makes the same codes operands again: a prompt of 8192 tokens 942 us; s c + b made in each tile 881, here 531 on one card and 564 on another (1035 and 975 TFLOP/s; a
// large matrix product has 1180). The price is a rounding of keys, values and weights to T: half a step each, as the reader's output and the result have it (weights in f16 down to
// 2^-25 of a row's largest).
//
// A workgroup has 16 MT rows for each of its waves, of one key head (new tokens times the query heads that share it), as columns of their matrix instructions, and goes through
// the tokens that they see 32 at a time. A block's keys and values come by load-to-LDS instructions, three stages of each, asked for two turns ahead; one barrier a turn.
// Workgroups of four waves, two to a compute unit, which go their own ways: one of eight has 614 us for that prompt, where this has 524. Rows of 48 to a wave (531), no scores ahead and
// three waves to a SIMD (521) and other orders of a turn's parts (524 - 535) are level.
#include "kv_attention.h"

namespace mtq {

namespace {

typedef _Float16 kv_f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t kv_f16_pair(uint32_t c1024, float s0, float s1, float b0, float b1) {   // (of 1024 + c, twice)
    const kv_f16x2 c = __builtin_bit_cast(kv_f16x2, c1024) - (kv_f16x2){(_Float16)1024.f, (_Float16)1024.f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, (kv_f16x2){(_Float16)s0, (_Float16)s1}, (kv_f16x2){(_Float16)b0, (_Float16)b1}));
}
template <int DT> __device__ __forceinline__ uint32_t kv_pack(float a, float b) {
    if constexpr (DT == DT_F16) {
        typedef __attribute__((ext_vector_type(2))) float f32x2;
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, kv_f16x2));
    } else {
        return kv_pack_bf16(a, b);
    }
}
// Codes as s c + b in T. bf16: f32 numbers, rounded by the pack; f16: c exactly, and one fused instruction's rounding.
template <int DT> struct Scale {   // of a word of codes of one group
    float s, b;
    __device__ __forceinline__ Scale(float s_, float b_) : s(s_), b(b_) {}
    __device__ __forceinline__ void word(uint32_t w, kr_u32x4& k) const {   // codes p and p + 4
        if constexpr (DT == DT_F16) {
#pragma unroll
            for (int p = 0; p < 4; p++) k[p] = kv_f16_pair((w >> (4 * p) & 0x000F000Fu) | 0x64006400u, s, s, b, b);
        } else {
            const uint32_t low = w & 0x0F0F0F0Fu, high = w >> 4 & 0x0F0F0F0Fu;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const uint32_t four = p & 1 ? high : low;
                k[p] = kv_pack_bf16(fmaf(s, (float)(four >> (p / 2 * 8) & 0xFFu), b), fmaf(s, (float)(four >> (16 + p / 2 * 8) & 0xFFu), b));
            }
        }
    }
};
template <int DT> struct Codes {   // a word of each of two tokens: of(e): both tokens' number e
    uint32_t w[2], low[2], high[2];
    float s[2], b[2];
    __device__ __forceinline__ Codes(uint32_t w0, uint32_t w1, float s0, float s1, float b0, float b1) : w{w0, w1}, low{w0 & 0x0F0F0F0Fu, w1 & 0x0F0F0F0Fu}, high{w0 >> 4 & 0x0F0F0F0Fu, w1 >> 4 & 0x0F0F0F0Fu}, s{s0, s1}, b{b0, b1} {}
    __device__ __forceinline__ uint32_t of(int e) const {
        if constexpr (DT == DT_F16) {
            const uint32_t two = __builtin_amdgcn_perm(w[1], w[0], 0x0C000C00u | (uint32_t)(4 + e / 2) << 16 | (uint32_t)(e / 2));
            return kv_f16_pair(((e & 1 ? two >> 4 : two) & 0x000F000Fu) | 0x64006400u, s[0], s[1], b[0], b[1]);
        } else {
            const uint32_t x = (e & 1 ? high[0] : low[0]) >> (e / 2 * 8) & 0xFFu, y = (e & 1 ? high[1] : low[1]) >> (e / 2 * 8) & 0xFFu;
            return kv_pack_bf16(fmaf(s[0], (float)x, b[0]), fmaf(s[1], (float)y, b[1]));
        }
    }
};

// A score at the bar weighs 2^LIFT, and the bar is raised when one passes it by 2^SLACK. f16 has its bits down to 2^-14 only and numbers up to 2^16: with 2^11 at the bar, weights
// down to 2^-25 of the largest are rounded by half a step of theirs (with 1 at the bar 12000 tokens of 2^-21.6 beside one whose value is 0 came out 3 % off, of 2^-24.5 44 %).
// A prompt of 8192 tokens has 563 us as before; 2^13 and 2^2 would take 573. bf16 has f32's exponents.
template <int DT> struct Weights {
    static constexpr float SLACK = DT == DT_F16 ? 4.f : kSlack, LIFT = DT == DT_F16 ? 11.f : 0.f;
};

template <int D> struct PromptShape {
    static constexpr int NW = D == 256 ? 8 : 4;                // waves of a workgroup
    static constexpr int MT = D == 256 ? 1 : 2;                // sixteens of rows of a wave
    static constexpr int STEPS = D / 32, NT = D / 16, ROWS = 16 * MT * NW;
    static constexpr int STAGE = kBlock * D * 2, STAGES = 3;   // of keys, or of values
    static constexpr int PER = STAGE / 1024 * 2 / NW;          // a wave's pieces of 1 KB of a block's keys, or of its values
    static constexpr uint32_t IMAGE = 2 * STAGE;
};

// Keys and values of 32 tokens of a sequence and key head by a wave: [keys][values], each as its stage has it.
template <int DT, int D, int G> __global__ __launch_bounds__(256) void kv_lay_kernel(KvAttentionArgs a, KvImages to) {
    using L = PromptShape<D>;
    constexpr int NG = D / G, STEPS = L::STEPS, KI = D / 64, VI = (D / 2 + 63) / 64;   // pieces of 32 codes of a token; of a word of eight tokens
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t head = blockIdx.x % kv.hkv, rest = blockIdx.x / kv.hkv, per = (to.blocks + 3u) / 4u, block = rest % per * 4u + wave;
    const KvSeq s = kv_seq(kv, rest / per);
    if (s.rows == 0 || kv.n_pages == 0 || block * kBlock >= s.len) return;
    const int32_t first = (int32_t)(s.len + 1u) - (int32_t)s.rows;   // what the first row sees: tokens up to here
    if (a.window && first > 0 && (uint32_t)first > a.window && (block + 1u) * kBlock <= (uint32_t)first - a.window) return;
    uint32_t slot[2], there = 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t at = block * kBlock + 16 * h, page = at < s.len ? kv.pages[(uint64_t)s.seq * kv.pages_stride + (at >> kv.page_log2)] : 0xFFFFFFFFu;
        // (of no page: one that is there. The pool has fewer than 2^32 tokens and heads: host)
        slot[h] = (((page < kv.n_pages ? page : 0u) * kv.hkv + head) << kv.page_log2) + (at & ((1u << kv.page_log2) - 1u));
        there |= page < kv.n_pages ? 1u << h : 0u;
    }
    const uint64_t index = ((uint64_t)s.seq * kv.hkv + head) * to.blocks + block;
    uint8_t* out = to.data + index * L::IMAGE;
    auto in = [&](uint32_t token) { return (there >> (token / 16) & 1u) && block * kBlock + token < s.len; };   // (where no token is: zeros)
    uint4 kw[KI];
    float ks[KI], kb[KI];
    uint32_t vw[VI][8];
    float vs[VI][8], vb[VI][8];
#pragma unroll
    for (int u = 0; u < KI; u++) {
        const uint32_t i = u * 64 + lane, token = i / 16 / STEPS * 16 + i % 16, step = i / 16 % STEPS, at = (token < 16 ? slot[0] : slot[1]) + token % 16;
        kw[u] = *(const uint4*)((const uint8_t*)kv.k.codes + (uint64_t)at * (D / 2) + step * 16);
        ks[u] = load_elem<DT>(kv.k.scales, (uint64_t)at * NG + step * 32 / G);
        kb[u] = load_elem<DT>(kv.k.biases, (uint64_t)at * NG + step * 32 / G);
    }
#pragma unroll
    for (int u = 0; u < VI; u++) {
        const uint32_t i = (u * 64 + lane) % (D / 2), quad = i / (D / 8), word = i % (D / 8);   // (of 64 numbers two lanes have the same)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t at = slot[j / 4] + 4 * quad + j % 4;
            vw[u][j] = *(const uint32_t*)((const uint8_t*)kv.v.codes + (uint64_t)at * (D / 2) + word * 4);
            vs[u][j] = load_elem<DT>(kv.v.scales, (uint64_t)at * NG + word * 8 / G);
            vb[u][j] = load_elem<DT>(kv.v.biases, (uint64_t)at * NG + word * 8 / G);
        }
    }
#pragma unroll
    for (int u = 0; u < KI; u++) {
        const uint32_t i = u * 64 + lane, token = i / 16 / STEPS * 16 + i % 16;
        const Scale<DT> sc(in(token) ? ks[u] : 0.f, in(token) ? kb[u] : 0.f);
        const uint32_t w[4] = {kw[u].x, kw[u].y, kw[u].z, kw[u].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            kr_u32x4 k;
            sc.word(w[j], k);
            *(kr_u32x4*)(out + (i / 16 * 64 + j * 16 + i % 16) * 16) = k;   // (i / 16: sixteen, then step)
        }
    }
    bool fine = true;
#pragma unroll
    for (int u = 0; u < VI; u++) {
        const uint32_t i = (u * 64 + lane) % (D / 2), quad = i / (D / 8), word = i % (D / 8);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool yes = in(j / 4 * 16 + 4 * quad + j % 4);
            vs[u][j] = yes ? vs[u][j] : 0.f;
            vb[u][j] = yes ? vb[u][j] : 0.f;
            fine = fine && fmaf(fabsf(vs[u][j]), 15.f, fabsf(vb[u][j])) < (DT == DT_F16 ? 65504.f : 3.38e38f);
        }
        const Codes<DT> two[4] = {Codes<DT>(vw[u][0], vw[u][1], vs[u][0], vs[u][1], vb[u][0], vb[u][1]), Codes<DT>(vw[u][2], vw[u][3], vs[u][2], vs[u][3], vb[u][2], vb[u][3]),
                                  Codes<DT>(vw[u][4], vw[u][5], vs[u][4], vs[u][5], vb[u][4], vb[u][5]), Codes<DT>(vw[u][6], vw[u][7], vs[u][6], vs[u][7], vb[u][6], vb[u][7])};
        uint8_t* at = out + L::STAGE + word / 2 * 1024 + (quad * 16 + word % 2 * 8) * 16;
#pragma unroll
        for (int e = 0; e < 8; e++) *(kr_u32x4*)(at + e * 16) = kr_u32x4{two[0].of(e), two[1].of(e), two[2].of(e), two[3].of(e)};
    }
    const bool all_fine = __all(fine);
    if (lane == 0) to.flags[index] = there | (all_fine ? 0u : 4u);
}

template <int DT, int D, int G>
__global__ __launch_bounds__(64 * PromptShape<D>::NW, 2) void kv_prompts_kernel(KvAttentionArgs a, KvParts parts, KvImages images, uint32_t tiles) {
    using L = PromptShape<D>;
    constexpr int NW = L::NW, MT = L::MT, NG = D / G, NT = L::NT, STEPS = L::STEPS, TH = 64 * NW, PER = L::PER;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const KvArgs& kv = a.kv;
    const uint32_t th = threadIdx.x, lane = th & 63u, wave = __builtin_amdgcn_readfirstlane(th >> 6), r = lane & 15u, g = lane >> 4;
    KvTile at_tile;
    if (!kv_tile<L::ROWS>(a, parts, tiles, at_tile)) return;
    const KvSeq& s = at_tile.s;
    const uint32_t shared = at_tile.shared, head = at_tile.head, rows = at_tile.rows, row0 = at_tile.row0, slice = at_tile.slice, slices = at_tile.slices;
    const uint32_t lo = at_tile.lo, hi = at_tile.hi, first_of_all = at_tile.first_end, b0 = at_tile.b0, b1 = at_tile.b1;
    auto end_of = [&](uint32_t i) { return kv_end(at_tile, i); };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    // This wave's rows, and a lane's.
    const uint32_t wave0 = row0 + wave * 16 * MT, wave_last = wave0 + 16 * MT - 1u < rows ? wave0 + 16 * MT - 1u : rows - 1u;
    const bool any = wave0 < rows;
    const uint32_t first_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave0) : 0u), last_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave_last) : 0u);
    const uint32_t last_from = from_of(last_end);
    uint32_t end[MT], from[MT];
    uint64_t row_at[MT];   // its row of the call
    uint32_t qh[MT];
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);   // (not 0: what is hidden scores -inf)
    kr_u32x4 q[MT][STEPS];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        uint32_t i = wave0 + 16 * m + r;
        if (i >= rows) i = rows - 1u;
        end[m] = end_of(i);
        from[m] = from_of(end[m]);
        row_at[m] = s.first_row + i / shared;
        qh[m] = head * shared + i % shared;
        const uint64_t q_at = row_at[m] * a.q_stride + (uint64_t)qh[m] * D + 8 * g;
#pragma unroll
        for (int j0 = 0; j0 < STEPS; j0++) {   // (values p and p + 4, as a word's codes come out)
            const kr_u32x4 v = *(const kr_u32x4*)((const uint16_t*)a.q + q_at + 32 * j0);
            const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
            for (int p = 0; p < 4; p++) q[m][j0][p] = __builtin_amdgcn_perm(v[2 + p / 2], v[p / 2], p & 1 ? 0x07060302u : 0x05040100u) ^ sign;
        }
    }

    // A block's keys or values into its stage: the first half of the waves has the keys.
    const bool values = wave >= NW / 2;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (values ? L::STAGES * L::STAGE : 0), piece = wave % (NW / 2) * PER;
    const uint64_t image0 = ((uint64_t)s.seq * kv.hkv + head) * images.blocks + lo / kBlock;   // of block 0
    const uint8_t* const image = images.data + image0 * L::IMAGE + (values ? L::STAGE : 0) + piece * 1024 + lane * 16;
    auto bring = [&](uint32_t b) {
        const uint32_t to = lds0 + b % L::STAGES * L::STAGE + piece * 1024;
        const uint8_t* from = image + (uint64_t)b * L::IMAGE;
#pragma unroll
        for (int u = 0; u < PER; u++) kv_load16(__builtin_amdgcn_readfirstlane(to + u * 1024), from + u * 1024);
    };
    // Until all of this wave's loads are there but those of the block asked for last (`behind`: it has been), and the others' as well.
    auto meet = [&](bool behind) {
        if (behind) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Flags of 64 blocks at a time, one to a lane (bits 0 and 1: a sixteen is on a page; 2: values that are no numbers).
    uint32_t flags = 0, flags_from = 0;
    auto flags_at = [&](uint32_t b) {
        flags_from = b;
        flags = b + lane < b1 ? images.flags[image0 + b + lane] : 0u;
    };
    auto flag = [&](uint32_t b) {
        if (b - flags_from > 63u) flags_at(b);
        return __builtin_amdgcn_readlane(flags, b - flags_from);
    };
    uint32_t* const none = (uint32_t*)(lds + 2 * L::STAGES * L::STAGE);   // a word for each group
    if (th < NG) none[th] = 0u;

    kr_f32x4 o[MT][NT] = {};
    float sum[MT] = {}, bar[MT];
    uint32_t poison = 0;   // (NG bits for each m: a group's values that are no numbers were seen)
#pragma unroll
    for (int m = 0; m < MT; m++) bar[m] = -INFINITY;
    // A sixteen of a block's keys, out of the LDS; and its scores.
    struct Keys {
        kr_u32x4 k[STEPS];
    };
    auto read_keys = [&](uint32_t b, int t, Keys& to) {
        const uint8_t* st = lds + b % L::STAGES * L::STAGE;
#pragma unroll
        for (int i = 0; i < STEPS; i++) to.k[i] = *(const kr_u32x4*)(st + (t * STEPS + i) * 1024 + lane * 16);
    };
    auto scores = [&](const Keys& from, int t, float (&x)[MT][2][4]) {
        kr_f32x4 acc[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) acc[m] = kr_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < STEPS; i++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[m] = kr_mfma<DT>(from.k[i], q[m][i], acc[m]);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[m][t][i] = acc[m][i];
    };
    // What a row does not see scores -inf; the bars are raised where scores pass them.
    uint32_t seen = 0xFFFFFFFFu;   // (8 bits for each m)
    bool whole = true, whole_of_all = true;   // (every row of the wave, and of the workgroup, sees all of the block)
    auto look = [&](uint32_t b, uint32_t there, float (&x)[MT][2][4]) {
        const uint32_t t0 = lo + b * kBlock;
        whole = t0 >= last_from && t0 + kBlock <= first_end && (there & 3u) == 3u;
        whole_of_all = t0 >= from_of(hi) && t0 + kBlock <= first_of_all && (there & 3u) == 3u;
        seen = 0xFFFFFFFFu;
        if (!whole) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t tok = t0 + 16 * t + 4 * g + i;
                        if (!((there >> t & 1u) && tok >= from[m] && tok < end[m])) {
                            x[m][t][i] = -INFINITY;
                            seen &= ~(1u << (8 * m + 4 * t + i));
                        }
                    }
        }
        float top[MT];
        bool over = false;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            top[m] = fmaxf(fmaxf(fmaxf(x[m][0][0], x[m][0][1]), fmaxf(x[m][0][2], x[m][0][3])), fmaxf(fmaxf(x[m][1][0], x[m][1][1]), fmaxf(x[m][1][2], x[m][1][3])));
            over = over || top[m] * c > bar[m] + Weights<DT>::SLACK;
        }
        if (__any(over)) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const float to = fmaxf(bar[m], kv_column_max(top[m]) * c), keep = to > bar[m] ? __builtin_amdgcn_exp2f(bar[m] - to) : 1.f;
                sum[m] *= keep;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[m][t][i] *= keep;
                bar[m] = to;
            }
        }
    };
    // A weight of 0 does not keep a NaN out: where some rows of the workgroup do not see all of a block, values that are no numbers
    // become zeros, and the rows that see them have a NaN in that group's sum.
    auto take_out = [&](uint32_t b) {
        uint8_t* st = lds + (L::STAGES + b % L::STAGES) * L::STAGE;
        constexpr uint32_t ALL = DT == DT_F16 ? 0x7C00u : 0x7F80u;   // an exponent of only ones
        for (uint32_t u = th; u < D / 16 * 64; u += TH) {
            uint16_t* p = (uint16_t*)(st + u / 64 * 1024 + u % 64 * 16);   // eight tokens' number 16 (u / 64) + u % 16
            uint32_t bad = 0;
            for (uint32_t j = 0; j < 8; j++)
                if ((p[j] & ALL) == ALL) {
                    p[j] = 0;
                    bad |= 1u << (j / 4 * 16 + u % 64 / 16 * 4 + j % 4);
                }
            if (bad) atomicOr(none + (u / 64 * 16 + u % 16) / G, bad);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const uint32_t bad = none[n];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if ((bad >> (16 * t + 4 * g + i) & 1u) && (seen >> (8 * m + 4 * t + i) & 1u)) poison |= 1u << (m * NG + n);
        }
        __syncthreads();
        if (th < NG) none[th] = 0u;
        __syncthreads();
    };
    // A block's weights out of its scores, one sixteen of them; a group's values and their numbers out of the LDS; p s as operands; and the values' sums.
    auto weigh = [&](int t, float (&x)[MT][2][4]) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float from_bar = bar[m] == -INFINITY ? 0.f : bar[m] - Weights<DT>::LIFT;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[m][t][i] = __builtin_amdgcn_exp2f(fmaf(x[m][t][i], c, -from_bar));
                sum[m] += x[m][t][i];
            }
        }
    };
    auto operands = [&](const float (&x)[MT][2][4], kr_u32x4 (&pt)[MT]) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < 4; j++) pt[m][j] = kv_pack<DT>(x[m][j / 2][2 * j % 4], x[m][j / 2][2 * j % 4 + 1]);
    };
    constexpr int PART = NT < 4 ? NT : 4;   // sixteens of numbers whose values are asked for together
    struct Values {
        kr_u32x4 v[PART];
    };
    auto read_values = [&](uint32_t b, int n, Values& to) {
        const uint8_t* st = lds + (L::STAGES + b % L::STAGES) * L::STAGE;
#pragma unroll
        for (int t = 0; t < PART; t++) to.v[t] = *(const kr_u32x4*)(st + (n * PART + t) * 1024 + lane * 16);
    };
    auto add_values = [&](const Values& from, int n, const kr_u32x4 (&pt)[MT]) {
#pragma unroll
        for (int t = 0; t < PART; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) o[m][n * PART + t] = kr_mfma<DT>(from.v[t], pt[m], o[m][n * PART + t]);
    };

    // The scores of a block are computed beside the values of the one before. In turn b the keys of block b + 3 and the values of b + 2 are asked for, into the
    // stages that turn b - 1 has read.
    if (b0 < b1) {
        float x[MT][2][4];
        const uint32_t ahead = values ? 2u : 3u;
        flags_at(b0);
        uint32_t now = flag(b0);
        bring(b0);
        if (b0 + 1u < b1) bring(b0 + 1u);
        if (!values && b0 + 2u < b1) bring(b0 + 2u);
        meet(b0 + ahead - 1u < b1);
        {
            Keys keys;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                read_keys(b0, t, keys);
                scores(keys, t, x);
            }
        }
        look(b0, now, x);
        meet(b0 + ahead - 1u < b1);
        for (uint32_t b = b0; b < b1; b++) {
            if (!whole_of_all && (now & 4u)) take_out(b);
            const uint32_t then = b + 1u < b1 ? flag(b + 1u) : 0u;
            if (b + ahead < b1) bring(b + ahead);
            // What the LDS is asked for in one part is used in the next (behind the last block the keys are those that are there, and not used).
            float next[MT][2][4];
            Keys first, second;
            Values group[2];
            kr_u32x4 pt[MT];
            read_keys(b + 1u, 0, first);
            weigh(0, x);
            __builtin_amdgcn_sched_barrier(0);
            read_keys(b + 1u, 1, second);
            scores(first, 0, next);
            weigh(1, x);
            __builtin_amdgcn_sched_barrier(0);
            read_values(b, 0, group[0]);
            scores(second, 1, next);
            operands(x, pt);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NT / PART; n++) {
                if (n + 1 < NT / PART) read_values(b, n + 1, group[(n + 1) & 1]);
                add_values(group[n & 1], n, pt);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (b + 1u < b1) look(b + 1u, then, next);
            now = then;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[m][t][i] = next[m][t][i];
            meet(b + ahead < b1);
        }
    }

#pragma unroll
    for (int m = 0; m < MT; m++) {
        const float total = kv_column_sum(sum[m]);
        const uint32_t i = wave0 + 16 * m + r;
        const uint64_t at = (row_at[m] * a.hq + qh[m]) * parts.slices + slice;
        if (parts.slices > 1 && i < rows && g == 0) {
            if (slices > 1) {
                parts.sums[at * 2] = bar[m];
                parts.sums[at * 2 + 1] = total;
            }
            const uint32_t n = slices == 1 ? 0u : slices;   // (of one slice: nothing to join)
            if (slice + 1u == slices && n < parts.slices) parts.sums[(at - slice + n) * 2 + 1] = kNoMore;
        }
        const float by = slices > 1 ? 1.f : total == 0.f ? 0.f : 1.f / total;
        uint32_t bad = poison >> (m * NG);
        bad |= (uint32_t)__shfl_xor((int)bad, 16, 64);
        bad |= (uint32_t)__shfl_xor((int)bad, 32, 64);
        if (i >= rows) continue;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const uint32_t d = 16 * t + 4 * g;
            const bool no_number = bad >> (16 * t / G) & 1u;
            kr_f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = no_number ? __builtin_nanf("") : slices == 1 && total == 0.f ? 0.f : o[m][t][j] * by;
            if (slices > 1) {
                *(kr_f32x4*)(parts.values + at * D + d) = v;
            } else {
                const uint64_t to = row_at[m] * a.out_stride + (uint64_t)qh[m] * D + d;
                *(uint2*)((uint16_t*)a.out + to) = make_uint2(kv_pack<DT>(v[0], v[1]), kv_pack<DT>(v[2], v[3]));
            }
        }
    }
}

template <int DT, int D, int G> int launch(const KvAttentionArgs& p, KvParts parts, KvImages images, const LaunchCtx& lc) {
    using L = PromptShape<D>;
    constexpr size_t LDS = 2 * L::STAGES * L::STAGE + D / G * 4;
    static_assert(LDS <= 160 * 1024, "");
    KvAttentionArgs a = p;
    const void *lay = (const void*)kv_lay_kernel<DT, D, G>, *fn = (const void*)kv_prompts_kernel<DT, D, G>;
    const uint64_t tiles64 = kv_sets<L::ROWS>(a);
    if (tiles64 * a.kv.hkv * parts.slices > max_workgroups(512)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    uint32_t tiles = (uint32_t)tiles64;
    LaunchCtx first = lc, second = lc, last = lc;
    first.stop = nullptr;
    second.start = nullptr;
    if (parts.slices > 1) second.stop = nullptr;
    last.start = nullptr;
    void* lay_args[] = {&a, &images};
    MTQ_HIP(launch_kernel(lay, dim3((images.blocks + 3) / 4 * a.kv.n_seqs * a.kv.hkv), dim3(256), lay_args, 0, first));
    MTQ_HIP(set_max_dynamic_lds(fn, LDS));
    void* args[] = {&a, &parts, &images, &tiles};
    MTQ_HIP(launch_kernel(fn, dim3(tiles * a.kv.hkv * parts.slices), dim3(64 * L::NW), args, LDS, second));
    return parts.slices > 1 ? launch_kv_join(DT, a, parts, last) : ERR_OK;
}

template <int DT> int launch_of(const KvAttentionArgs& p, const KvParts& parts, const KvImages& images, const LaunchCtx& lc) {
    switch (p.kv.dim * 1000 + p.kv.group) {
        case 64032: return launch<DT, 64, 32>(p, parts, images, lc);
        case 64064: return launch<DT, 64, 64>(p, parts, images, lc);
        case 128032: return launch<DT, 128, 32>(p, parts, images, lc);
        case 128064: return launch<DT, 128, 64>(p, parts, images, lc);
        case 128128: return launch<DT, 128, 128>(p, parts, images, lc);
        case 256032: return launch<DT, 256, 32>(p, parts, images, lc);
        case 256064: return launch<DT, 256, 64>(p, parts, images, lc);
        case 256128: return launch<DT, 256, 128>(p, parts, images, lc);
    }
    return fail(ERR_UNSUPPORTED, "kv_attention: no kernel for this head_dim and group_size");
}

}  // namespace

int launch_kv_prompts(int dtype, const KvAttentionArgs& p, const KvParts& parts, const KvImages& images, const LaunchCtx& lc) {
    return dtype == DT_F16 ? launch_of<DT_F16>(p, parts, images, lc) : launch_of<DT_BF16>(p, parts, images, lc);
}

// Rows of a tile, by which the slices are chosen.
uint32_t kv_prompt_rows(uint32_t dim) { return dim == 256 ? PromptShape<256>::ROWS : PromptShape<128>::ROWS; }

}  // namespace mtq
