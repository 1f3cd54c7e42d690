// What both attention kernels over the 4-bit cache have in common.
//
//   out = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  k_j = s c + b and v_j = s c + b with codes c in 0..15 and s, b of a token and group
//
// Codes are operands of the matrix instructions as they are: a nibble in the mantissa of 16 is the number 16 + c, in bf16 (bits 3..6) and in f16 (bits
// 6..9), one mask and one OR for two of them. What that adds is taken out in f32:
//   scores  s sum_d q (16 + c) + (b - 16 s) sum_d q, for each group
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
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ float kv_column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// What joins the parts of a row: the maximum in base 2, the sum of the weights, and the weighted values, rows of dim.
struct KvParts {
    float* values = nullptr;   // [rows, query heads, slices, dim]
    float* sums = nullptr;     // [rows, query heads, slices, 2]
    uint32_t slices = 1;
};
int launch_kv_rows(int dtype, const KvAttentionArgs& p, const KvParts& parts, bool large, const LaunchCtx& lc);
int launch_kv_tiles(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
int launch_kv_join(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc);
uint32_t kv_tile_rows(int dtype, uint32_t dim);

}  // namespace mtq
