// Few activation rows times a weight matrix in 8-bit floating point (fp8_common.h): bound by the one read of the weights.
//
//   out[m, n] = sum over blocks b of xs[m, b] ws[n / 128, b] (sum over b's k of x[m, k] w[n, k])
//
// The inner sum is one 16 x 16 x 128 matrix instruction; its two scales differ by block and by row of the
// result, so they are multiplied in behind it, one f32 FMA a value. A workgroup has 16 weight rows, whose blocks its waves share;
// the weights go from memory to the matrix cores' registers, eight lines of 16 rows in flight a wave.
#include "fp8_common.h"

namespace mtq {

namespace {

constexpr int kFp8Depth = 4;   // blocks of a wave's rows in flight

// MT: 16-row blocks of activations (codes); NW: waves.
template <int DT, int MT, int NW> __global__ __launch_bounds__(64 * NW) void fp8_rows_kernel(Fp8Args a) {
    __shared__ fp8_f32x4 part[NW][MT][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    const uint32_t r = lane & 15u, g = lane >> 4, blocks = (a.K + kFp8Block - 1) / kFp8Block;
    const uint32_t n = n0 + r < a.N ? n0 + r : a.N - 1;
    const uint8_t* w = a.w + (size_t)n * a.K + 16 * g;
    const float* ws = a.ws + (size_t)(n0 / kFp8Block) * blocks;
    const uint8_t* x[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const uint32_t m = m0 + 16 * t + r;
        x[t] = (const uint8_t*)a.x + (size_t)(m < a.M ? m : a.M - 1) * a.K + 16 * g;
    }
    fp8_f32x4 acc[MT] = {};
    for (uint32_t b0 = wave; b0 < blocks; b0 += NW * kFp8Depth) {
        uint4 wv[kFp8Depth][2];
#pragma unroll
        for (int d = 0; d < kFp8Depth; d++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t k = (b0 + d * NW) * kFp8Block + 64 * h;
                wv[d][h] = k + 16 * g < a.K ? *(const uint4*)(w + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int d = 0; d < kFp8Depth; d++) {
            const uint32_t b = b0 + d * NW;
            if (b >= blocks) break;
            const float sw = ws[b];
#pragma unroll
            for (int t = 0; t < MT; t++) {
                uint4 xv[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t k = b * kFp8Block + 64 * h;
                    xv[h] = k + 16 * g < a.K ? *(const uint4*)(x[t] + k) : make_uint4(0, 0, 0, 0);
                }
                const fp8_f32x4 p = fp8_mfma<DT>(xv[0], xv[1], wv[d][0], wv[d][1]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t m = m0 + 16 * t + 4 * g + i;
                    const float sx = a.xs[(size_t)(m < a.M ? m : a.M - 1) * blocks + b];
                    acc[t][i] += p[i] * (sx * sw);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (uint32_t t = wave; t < MT; t += NW) {
        fp8_f32x4 sum = part[0][t][lane];
        for (int v = 1; v < NW; v++) sum += part[v][t][lane];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t m = m0 + 16 * t + 4 * g + i;
            if (m < a.M && n0 + r < a.N) store_elem<DT>(a.out, (size_t)m * a.N + n0 + r, sum[i]);
        }
    }
}

template <int DT> const void* rows_fn(int mt) {
    return mt == 1 ? (const void*)fp8_rows_kernel<DT, 1, 4> : mt == 2 ? (const void*)fp8_rows_kernel<DT, 2, 4> : (const void*)fp8_rows_kernel<DT, 4, 4>;
}

}  // namespace

int launch_fp8_rows(int dtype, const Fp8Args& p, const LaunchCtx& lc) {
    Fp8Args a = p;
    const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const uint32_t ny = (a.M + 16 * mt - 1) / (16 * mt);
    if (ny > 65535u) return fail(ERR_SHAPE, "too many activation rows");
    const void* fn = dtype == DT_F32 ? rows_fn<DT_F32>(mt) : dtype == DT_F16 ? rows_fn<DT_F16>(mt) : rows_fn<DT_BF16>(mt);
    void* args[] = {&a};
    MTQ_HIP(launch_kernel(fn, dim3((a.N + 15) / 16, ny), dim3(256), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
