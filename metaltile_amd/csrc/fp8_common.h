// 8-bit floating point in blocks of 128: codes are e4m3 (OCP: four exponent and three mantissa bits, largest 448), row-major bytes, and a
// block of codes has one f32 scale. value = code * scale, scale = max |x| / 448 over the block (1 for a block of zeros). Activations have
// blocks of 1 x 128 (scales [rows, ceil(K / 128)]), weights of 128 x 128 ([ceil(N / 128), ceil(K / 128)]); blocks at the far edges may be cut.
#pragma once
#include "mtq_device.h"
#include "mtq_internal.h"

namespace mtq {

constexpr uint32_t kFp8Block = 128;
constexpr float kFp8Most = 448.f;
constexpr uint32_t kFp8TilesLongest = 1u << 22;   // K up to which a tile's rows have 31-bit offsets

typedef int fp8_i32x8 __attribute__((ext_vector_type(8)));
typedef float fp8_f32x4 __attribute__((ext_vector_type(4)));

// Eight elements from p[i ..], in f32 (i * element size a multiple of 16 bytes).
template <int DT> __device__ __forceinline__ void fp8_load8(const void* p, size_t i, float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 r = *(const uint4*)((const uint16_t*)p + i);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
            v[j] = DT == DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}

// The larger magnitude; what is no number counts as nothing (its code is NaN under any scale).
__device__ __forceinline__ float fp8_most(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[j]));
    return m;
}
__device__ __forceinline__ float seg16_max(float v) {   // over rows of 16 lanes, v >= 0
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x141>(v));
    return fmaxf(v, dpp_f32<0x140>(v));
}
__device__ __forceinline__ float fp8_scale(float most) { return most > 0.f ? fmaxf(most / kFp8Most, 1.17549435e-38f) : 1.f; }

// Codes of eight elements: the quotient by the scale in f32 (correctly rounded), then the nearest e4m3 value, ties to even.
// A division is a dozen instructions, which is more than memory leaves time for (4096 x 4096 bf16 by rows: 13.2 us, 10.6 without). With r the
// correctly rounded 1 / scale, v r is within 1.5 ulp of the quotient; a step q + r (v - q scale) makes it one of the two nearest, and a
// second the nearest (Markstein's theorem: the difference is exact, and no quotient is closer to the middle of two f32 than the error that is
// left). That holds while nothing underflows: a quotient that rounds to more than zero is 2^-10 or more, and the difference a multiple of 2^-47
// of v = 2^-10 scale: scales of 2^-80 and more leave it in range, others are divided by (a scale that is infinite, too).
__device__ __forceinline__ uint2 fp8_codes(const float (&v)[8], float scale) {
    float q[8];
    if (scale >= 8.27180613e-25f && scale < INFINITY) {
        const float r = 1.f / scale;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            q[j] = v[j] * r;
            q[j] = fmaf(fmaf(-q[j], scale, v[j]), r, q[j]);
            q[j] = copysignf(fmaf(fmaf(-q[j], scale, v[j]), r, q[j]), v[j]);   // (of zeros the sums lose the sign)
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = v[j] / scale;
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// 16 x 16 x 128 on the matrix cores, from zero: a lane gives 32 bytes of row lane & 15 of either operand. Which 32 of the 128 is the same
// choice for both (bytes 16 g .. and 64 + 16 g .. for g = lane >> 4, so that four lanes read whole lines), and the sum does not depend on it.
// Result: column lane & 15 (of b's rows), rows 4 (lane >> 4) + i (of a's).
// The instruction on 8-bit operands lines up the products of eight neighbouring codes by the largest of them and drops what lies below
// 2^-13 of its power of two (measured: 2^16 + 2^3 is kept, 2^16 + 2^2 is not), then sums in f32: about 1e-5 of a result whose terms have
// no order, a fiftieth of an f16 rounding and a four-hundredth of a bf16 one. Results in f32 take the same codes as bf16 operands
// (e4m3 values are bf16 values), whose products and sums keep 24 bits, at half the rate.
template <int DT> __device__ __forceinline__ fp8_f32x4 fp8_mfma(uint4 a0, uint4 a1, uint4 b0, uint4 b1) {
    const fp8_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DT == DT_F32) {
        typedef __attribute__((ext_vector_type(8))) __bf16 v8;
        const uint32_t a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
        auto wide = [](uint32_t lo, uint32_t hi) {
            const auto p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
            const auto r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
            return v8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
        };
        fp8_f32x4 c = zero;
#pragma unroll
        for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide(a[i], a[i + 1]), wide(b[i], b[i + 1]), c, 0, 0, 0);
        return c;
    } else {
        const fp8_i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
        const fp8_i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);
    }
}

__device__ __host__ __forceinline__ uint32_t fp8_blocks(uint32_t k) { return (k >> 7) + ((k & 127u) != 0); }

// Four neighbouring results of row m, n a multiple of 4.
template <int DT> __device__ __forceinline__ void fp8_store4(void* out, uint32_t m, uint32_t n, uint32_t N, fp8_f32x4 v) {
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const size_t i0 = (size_t)m * N + n;
    if (N % 4 == 0 && (uintptr_t)out % (4 * ES) == 0 && n < N) {
        if constexpr (DT == DT_F32) {
            *(fp8_f32x4*)((float*)out + i0) = v;
        } else {
            *(uint2*)((uint16_t*)out + i0) = make_uint2(f32_to_elem_bits<DT>(v[0]) | (uint32_t)f32_to_elem_bits<DT>(v[1]) << 16,
                                                        f32_to_elem_bits<DT>(v[2]) | (uint32_t)f32_to_elem_bits<DT>(v[3]) << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n + i < N) store_elem<DT>(out, i0 + i, v[i]);
    }
}

// Tile i of the n in a launch: workgroups go to the eight XCDs in turn, and each XCD gets a run of neighbours.
__device__ __forceinline__ uint32_t xcd_run(uint32_t i, uint32_t n) {
    const uint32_t per = n / 8, extra = n % 8, xcd = i % 8;
    return xcd * per + (xcd < extra ? xcd : extra) + i / 8;
}

struct Fp8Args {
    const uint8_t* w;      // codes [N, K]
    const float* ws;       // [ceil(N / 128), ceil(K / 128)]
    const void* x;         // codes [M, K], or T [M, K] that the kernel quantises
    const float* xs;       // [M, ceil(K / 128)] (codes)
    void* out;             // T [M, N]
    uint32_t M, N, K;
};

inline int fp8_num_cus() {
    static int n = 0;
    if (n == 0) {
        int dev = 0, v = 0;
        n = (hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) ? v : 256;
    }
    return n;
}

}  // namespace mtq
