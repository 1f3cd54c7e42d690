// What the attention kernels over the 4-bit cache have in common.
//
//   out = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  k_j = s c + b and v_j = s c + b with codes c in 0..15 and s, b of a token and group
//
// Codes are operands of the matrix instructions as they are: a nibble in the mantissa of 16 is the number 16 + c, in bf16 (bits 3..6) and in f16 (bits
// 6..9), one mask and one OR for two of them. What that adds is taken out in f32:
//   scores  s sum_d q (16 + c) + (b - 16 s) sum_d q, for each group (or s (sum_d q (16 + c) - 16 sum_d q) + b sum_d q)
//   values  sum_j (p s) (16 + c) - 24 sum_j (p s) + sum_j p (b + 8 s), where the first two sums have the same rounded p s, so that its rounding
//           meets c - 8, a code's distance from the middle, and the last is f32
// p s is rounded to bf16 for bf16 (half a step, as the result is), and is two or three bf16 terms for f16 and f32; an f32 query is three terms.
// A score's instruction has tokens as rows and queries as columns, so a lane ends up with four neighbouring tokens of one query, which is what the
// values' instruction wants of p: the tokens of its sum are taken in that order, and nothing goes between lanes. The softmax is in base 2, and
// relative to a bar that is raised only when a score passes it by 2^kSlack: until then there is nothing to exchange and nothing to rescale.
#pragma once
#include "kv_cache.h"
#include "mfma16.h"

namespace mtq {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kSlack = 8.f;

template <int DT> struct KvTerms {
    static constexpr int Q = DT == DT_F32 ? 3 : 1;                          // terms of a query
    static constexpr int P = DT == DT_F32 ? 3 : DT == DT_F16 ? 2 : 1;       // bf16 terms of p s
    static constexpr int QK = DT == DT_F16 ? DT_F16 : DT_BF16;              // the scores' operands
    static constexpr bool CENTRED = DT == DT_F32;                           // operands are c - 8, not 16 + c
};

// Nibbles `p` and p + 4 of a word as 16 + c, in the lower and the upper half. `base` is 16 twice, in a vector register (one mask and OR then).
template <int QK> __device__ __forceinline__ uint32_t kv_sixteen() {
    uint32_t k = QK == DT_BF16 ? 0x41804180u : 0x4C004C00u;
    asm volatile("" : "+v"(k));
    return k;
}
template <int QK> __device__ __forceinline__ uint32_t kv_pair(uint32_t w, int p, uint32_t base) {
    const int up = (QK == DT_BF16 ? 3 : 6) - 4 * p;
    return ((up >= 0 ? w << up : w >> -up) & (QK == DT_BF16 ? 0x00780078u : 0x03C003C0u)) | base;
}

// f32 takes c - 8: of 16 + c the sums are four times as large, and what they lose by it was most of its error (of 1000 tokens 2.6e-6 of the result).
template <int DT> __device__ __forceinline__ uint32_t kv_operand(uint32_t pair) {
    if constexpr (!KvTerms<DT>::CENTRED) return pair;
    const float low = __uint_as_float(pair << 16) - 24.f, high = __uint_as_float(pair & 0xFFFF0000u) - 24.f;
    return __builtin_amdgcn_perm(__float_as_uint(high), __float_as_uint(low), 0x07060302u);   // (exact in bf16)
}

// An f32 value in bf16 terms.
template <int N> __device__ __forceinline__ void kv_split(float v, float (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        t[i] = i + 1 < N ? bf16_bits_to_f32(f32_to_elem_bits<DT_BF16>(v)) : v;   // (the last is rounded where it is packed)
        v -= t[i];
    }
}
__device__ __forceinline__ uint32_t kv_pack_bf16(float a, float b) {   // (one instruction as a vector of two, four as two numbers)
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2_t));
}

// Sum and maximum over the lanes of a column (lane & 15).
__device__ __forceinline__ float kv_column_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float kv_column_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// SIZE bytes a lane from `from` to LDS: lane l's at lds + SIZE l. No register is written; counts in vmcnt. M0 is read one wait state behind its write at
// the earliest, which no one but this block sees to.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // M0 is a reserved register: naming it as clobbered is the point
__device__ __forceinline__ void kv_load16(uint32_t lds, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void kv_load4(uint32_t lds, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// What joins the parts of a row: the maximum in base 2, the sum of the weights, and the weighted values, rows of dim.
struct KvParts {
    float* values = nullptr;   // [rows, query heads, slices, dim]
    float* sums = nullptr;     // [rows, query heads, slices, 2]; a sum of -1 (kNoMore): no slice from here on
    uint32_t slices = 1;       // that a sequence has at most
    uint32_t pieces = 1;       // of the kernels for few rows: what all sequences' tokens are cut into, about (kv_piece)
    uint32_t least = 1;        // blocks of 64 tokens that a piece has
};
constexpr float kNoMore = -1.f;
constexpr uint32_t kCutSeqs = 512;   // sequences that are cut into pieces at most: each workgroup looks at all of them

// The sum of this lane's value and those of the lanes below.
__device__ __forceinline__ uint32_t kv_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);   // (1, 2, 4 and 8 lanes below in the sixteen; nothing where there are none)
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);   // (the last of the sixteen below, then of the half)
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}

// Rows of a sequence and key head (new tokens times the query heads that share it) go to workgroups in sets of ROWS. Sequence i's sets begin at
// (its first row * shared + i * loose) / ROWS, loose = ROWS - the largest power of two in `shared` up to ROWS: a sequence's rows are whole multiples of that, so there is room for
// as many sets as it has, and often for no more.
template <uint32_t ROWS> __host__ __device__ inline uint32_t kv_loose(uint32_t shared) {
    const uint32_t g = shared & (0u - shared);
    return g < ROWS ? ROWS - g : 0u;
}
template <uint32_t ROWS> inline uint64_t kv_sets(const KvAttentionArgs& a) {   // that there is room for
    const uint32_t shared = a.hq / a.kv.hkv;
    return ((uint64_t)a.kv.n_tokens * shared + (uint64_t)a.kv.n_seqs * kv_loose<ROWS>(shared)) / ROWS;
}
// The sequence that set `index` lies in, and which of its sets it is. False: none. All lanes of a wave call.
template <uint32_t ROWS> __device__ __forceinline__ bool kv_find(const KvAttentionArgs& a, uint32_t index, KvSeq& s, uint32_t& set) {
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u, shared = a.hq / kv.hkv, loose = kv_loose<ROWS>(shared);
    auto begin = [&](uint32_t first_row, uint32_t i) { return (uint32_t)(((uint64_t)first_row * shared + (uint64_t)i * loose) / ROWS); };
    uint32_t seq;
    if (kv.offsets) {
        uint32_t lo = 0, n = kv.n_seqs;   // of the sequences lo .. lo + n - 1 the last that begins at `index` or before
        while (n > 1) {
            const uint32_t step = (n + 63u) / 64u, i = lo + lane * step;
            const bool before = lane * step < n && begin(kv.offsets[i] < kv.n_tokens ? kv.offsets[i] : kv.n_tokens, i) <= index;
            const uint32_t count = (uint32_t)__popcll(__ballot(before));
            const uint32_t skip = count ? (count - 1u) * step : 0u;
            lo += skip;
            n = n - skip < step ? n - skip : step;
        }
        seq = __builtin_amdgcn_readfirstlane(lo);
    } else {
        const uint32_t rows = kv.n_tokens / kv.n_seqs;   // (the last i with begin(i rows, i) <= index)
        const uint64_t per = (uint64_t)rows * shared + loose, i = per ? (uint64_t)index * ROWS / per : 0u;
        seq = (uint32_t)(i < kv.n_seqs ? i : kv.n_seqs - 1u);
        while (seq + 1u < kv.n_seqs && begin((seq + 1u) * rows, seq + 1u) <= index) seq++;
    }
    s = kv_seq(kv, seq);
    const uint32_t first = begin(s.first_row, seq);
    set = index - first;
    return index >= first && (uint64_t)set * ROWS < (uint64_t)s.rows * shared;
}

// Workgroup `index` of a key head's: a sequence's set of rows, and one of the equal slices that its tokens are cut into. Lengths are known here only, and sequences of
// 1 to 8192 tokens, each cut into as many, left the card with the longest one's slices: so a piece is a share of all tokens, and a sequence has as many as its
// tokens need. False: no piece. All lanes of a wave call.
struct KvPiece {
    KvSeq s;
    uint32_t set = 0, slice = 0, slices = 1;
};
template <uint32_t ROWS, uint32_t EACH> __device__ __forceinline__ bool kv_piece_of(const KvAttentionArgs& a, const KvParts& parts, uint32_t index, KvPiece& p) {   // EACH sequences to a lane
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u, each = EACH == 1 ? 1u : (kv.n_seqs + 63u) / 64u, shared = a.hq / kv.hkv;
    KvSeq s[EACH];
    uint32_t n[EACH], sets[EACH], all = 0;   // their blocks of 64 tokens
    auto from_of = [&](uint32_t j) {         // what the first row sees first
        const int32_t end = (int32_t)(s[j].len + 1u) - (int32_t)s[j].rows;
        return a.window && end > 0 && (uint32_t)end > a.window ? (uint32_t)end - a.window : 0u;
    };
#pragma unroll
    for (uint32_t j = 0; j < EACH; j++) {
        const uint32_t i = lane * each + j;
        s[j] = KvSeq{0, 0, 0, 0};
        if (j < each && i < kv.n_seqs) s[j] = kv_seq(kv, i);
        sets[j] = (s[j].rows * shared + ROWS - 1u) / ROWS;
        n[j] = (s[j].len - from_of(j) + 63u) / 64u;
        all += n[j] * sets[j];
    }
    uint32_t share = ((uint32_t)__builtin_amdgcn_readlane((int)kv_scan(all), 63) + parts.pieces - 1u) / parts.pieces;
    if (share < parts.least) share = parts.least;
    // Those whose pieces are nearest to a share come first, in four classes, so that a compute unit gets long, middling and short ones alike (64 sequences of 1 to 8192
    // tokens: 72 us, in their own order 81).
    uint32_t class_of[EACH], mine[4] = {};
#pragma unroll
    for (uint32_t j = 0; j < EACH; j++) {
        const uint32_t whole = n[j];
        n[j] = whole <= share ? 1u : (whole + share - 1u) / share;
        if (n[j] > parts.slices) n[j] = parts.slices;
        const uint64_t eights = (uint64_t)(n[j] == 1u ? whole : (whole + n[j] - 1u) / n[j]) * 8u;
        class_of[j] = eights > share * 7ull ? 0u : eights > share * 5ull ? 1u : eights > share * 3ull ? 2u : 3u;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) mine[i] += class_of[j] == i ? n[j] * sets[j] : 0u;
    }
    uint32_t before = 0, rest = 0, in = 4;   // (this lane's answer; `who` has the one that counts)
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t upto = kv_scan(mine[i]), begin = before + upto - mine[i];
        if (index - begin < mine[i]) {
            rest = index - begin;
            in = i;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    const uint64_t his_is = __ballot(in < 4u);
    if (!his_is) return false;
    const int who = __builtin_ctzll(his_is);
    uint32_t slices = 1, of = 1;
    KvSeq found = s[0];
    bool yes = false;
#pragma unroll
    for (uint32_t j = 0; j < EACH; j++)
        if (!yes && class_of[j] == in) {
            if (rest < n[j] * sets[j]) {
                yes = true;
                found = s[j];
                slices = n[j];
                of = sets[j];
            } else {
                rest -= n[j] * sets[j];
            }
        }
    auto his = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, who); };
    p.s = KvSeq{his(found.seq), his(found.first_row), his(found.rows), his(found.len)};
    rest = his(rest);
    of = his(of);
    p.slice = rest / of;
    p.set = rest - p.slice * of;
    p.slices = his(slices);
    return true;
}
template <uint32_t ROWS> __device__ __forceinline__ bool kv_piece(const KvAttentionArgs& a, const KvParts& parts, uint32_t index, KvPiece& p) {
    if (parts.slices > 1) return a.kv.n_seqs <= 64 ? kv_piece_of<ROWS, 1>(a, parts, index, p) : kv_piece_of<ROWS, kCutSeqs / 64>(a, parts, index, p);
    return kv_find<ROWS>(a, index, p.s, p.set);
}

constexpr uint32_t kBlock = 32;   // tokens of a step of the kernels for many rows
// A workgroup of those: ROWS rows of a key head (new tokens times the query heads that share it), and blocks b0 .. b1 - 1 of the tokens that they see.
struct KvTile {
    KvSeq s;
    uint32_t head, shared, rows, row0, slice, slices;   // row0 .. row0 + ROWS - 1 of the sequence's `rows`
    uint32_t lo, hi, first_end, b0, b1;                 // they see tokens lo (of block 0) .. hi - 1; its first row those below first_end
};
template <uint32_t ROWS> __device__ __forceinline__ bool kv_tile(const KvAttentionArgs& a, const KvParts& parts, uint32_t tiles, KvTile& to) {
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t shared = a.hq / kv.hkv, head = blockIdx.x % kv.hkv, at_tile = blockIdx.x / kv.hkv, slice = at_tile / tiles;
    KvSeq s;
    uint32_t set;
    if (!kv_find<ROWS>(a, tiles - 1u - at_tile % tiles, s, set)) return false;   // (the last ones see the most and come first)
    const uint32_t rows = s.rows * shared, row0 = set * ROWS;

    auto end_of = [&](uint32_t i) { const int32_t e = (int32_t)(s.len + i / shared + 1u) - (int32_t)s.rows; return e > 0 ? (uint32_t)e : 0u; };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    const uint32_t last = row0 + ROWS - 1u < rows ? row0 + ROWS - 1u : rows - 1u;
    const uint32_t hi = __builtin_amdgcn_readfirstlane(end_of(last)), first_of_all = __builtin_amdgcn_readfirstlane(end_of(row0)), lo = __builtin_amdgcn_readfirstlane(from_of(end_of(row0))) & ~31u;
    const uint32_t blocks = kv.n_pages && hi > lo ? (hi - lo + kBlock - 1u) / kBlock : 0u;
    // A tile is cut into slices by what it sees, against what all see: of a prompt its last tiles, of several the longest one's.
    uint32_t slices = 1;
    if (parts.slices > 1) {
        uint32_t all = 0;   // blocks that tiles see, as many or a few more
        for (uint32_t i = lane; i < kv.n_seqs; i += 64) {
            const KvSeq o = kv_seq(kv, i);
            const uint32_t n = (o.rows * shared + ROWS - 1u) / ROWS, before = o.len > o.rows ? o.len - o.rows : 0u;
            uint32_t mean = (before + o.len + ROWS / shared + 1u) / 2u;
            if (a.window && mean > a.window + ROWS / shared) mean = a.window + ROWS / shared;
            all += n * (mean / kBlock + 1u);
        }
        for (int i = 1; i < 64; i <<= 1) all += (uint32_t)__shfl_xor((int)all, i, 64);
        uint32_t share = (all + parts.pieces - 1u) / parts.pieces;
        if (share < parts.least) share = parts.least;
        slices = __builtin_amdgcn_readfirstlane((blocks + share - 1u) / share);
        if (slices > parts.slices) slices = parts.slices;
        if (slices < 1u) slices = 1u;
        if (slice >= slices) return false;
    }
    const uint32_t per = (blocks + slices - 1u) / slices;
    const uint32_t b0 = slice * per < blocks ? slice * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
    to = KvTile{s, head, shared, rows, row0, slice, slices, lo, hi, first_of_all, b0, b1};
    return true;
}
__device__ __forceinline__ uint32_t kv_end(const KvTile& t, uint32_t i) {   // row i sees the tokens before this one
    const int32_t e = (int32_t)(t.s.len + i / t.shared + 1u) - (int32_t)t.s.rows;
    return e > 0 ? (uint32_t)e : 0u;
}
// Workgroups of a key head: pieces there can be.
template <uint32_t ROWS> inline uint64_t kv_pieces(const KvAttentionArgs& a, const KvParts& parts) { return kv_sets<ROWS>(a) + (parts.slices == 1 ? 0u : parts.pieces); }
int launch_kv_rows(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
int launch_kv_quads(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
int launch_kv_tiles(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
// Keys and values of 32 tokens in T, as the matrix instructions take them (kv_attention_prompts.hip).
struct KvImages {
    uint8_t* data = nullptr;     // [sequences, key heads, blocks], 128 head_dim bytes each
    uint32_t* flags = nullptr;   // [sequences, key heads, blocks]
    uint32_t blocks = 0;         // of a sequence
};
int launch_kv_prompts(int dtype, const KvAttentionArgs& p, const KvParts& parts, const KvImages& images, const LaunchCtx& lc);
uint32_t kv_prompt_rows(uint32_t dim);
int launch_kv_join(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
uint32_t kv_tile_rows(int dtype, uint32_t dim);

}  // namespace mtq
