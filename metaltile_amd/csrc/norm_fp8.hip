// Residual addition, RMS norm and quantising into 8-bit floating point (fp8_common.h), in one read of the rows and one write of the sums and codes.
//   h = x + r,  y = (h w) / sqrt(sum h^2 / cols + eps),  a scale and codes of y for each 128 of a row
// Bound by memory; the rows of a decode step by latency. A row stays in registers between its sum of squares and its codes, eight elements a lane
// and 16 lanes a block of 128, as in the quantiser. Rows of more than 65536 elements are read again.
#include "fp8_common.h"

namespace mtq {

namespace {

// PAST: past the caches, from kLarge elements on, where what is written would push out what is still read (5000 x 4144 f16: 32 us against 38).
constexpr uint64_t kLarge = 1ull << 23;
template <int N, bool PAST> __device__ __forceinline__ void norm_put(void* p, const uint32_t (&w)[N]) {
    typedef uint32_t vec __attribute__((ext_vector_type(N)));
    vec v;
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = w[j];
    if constexpr (PAST) __builtin_nontemporal_store(v, (vec*)p);
    else *(vec*)p = v;
}
template <int DT, bool PAST> __device__ __forceinline__ void norm_store8(void* p, size_t i, const float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        norm_put<4, PAST>((float*)p + i, {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
        norm_put<4, PAST>((float*)p + i + 4, {__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t)f32_to_elem_bits<DT>(v[2 * j]) | (uint32_t)f32_to_elem_bits<DT>(v[2 * j + 1]) << 16;
        norm_put<4, PAST>((uint16_t*)p + i, w);
    }
}

// T threads a row, V vectors of eight a thread held in registers; V 0: any length, read twice. Workgroups of max(T, 256) threads.
template <int DT, int T, int V, bool PAST> __global__ __launch_bounds__(T < 256 ? 256 : T) void norm_fp8_kernel(NormFp8Args a) {
    constexpr int ROWS = T < 256 ? 256 / T : 1, HELD = V ? V : 1, AHEAD = V <= 2 ? HELD : 0;   // (AHEAD: vectors of weights that there is room for)
    __shared__ float part[T / 64 ? T / 64 : 1];
    const uint32_t tid = threadIdx.x % T, row = blockIdx.x * ROWS + threadIdx.x / T;
    if (row >= a.rows) return;   // (whole waves, and of a row with several all of them)
    const size_t at = (size_t)row * a.cols;
    const uint32_t blocks = fp8_blocks(a.cols);
    auto sum8 = [&](uint32_t col, float (&h)[8]) {
        fp8_load8<DT>(a.x, at + col, h);
        if (a.residual) {
            float r[8];
            fp8_load8<DT>(a.residual, at + col, r);
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] += r[j];
        }
    };
    float h[HELD][8] = {}, weights[AHEAD ? AHEAD : 1][8] = {}, ssq = 0.f;   // (the weights are asked for with the row: one way from memory, not two)
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = (i * T + tid) * 8;
            if (col < a.cols) {
                sum8(col, h[i]);
                if constexpr (AHEAD) fp8_load8<DT>(a.weight, col, weights[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) ssq = fmaf(h[i][j], h[i][j], ssq);
    } else {
        for (uint32_t col = tid * 8; col < a.cols; col += T * 8) {
            sum8(col, h[0]);
#pragma unroll
            for (int j = 0; j < 8; j++) ssq = fmaf(h[0][j], h[0][j], ssq);
        }
    }
    ssq = seg_allreduce(ssq, 64);
    if constexpr (T > 64) {
        if ((tid & 63u) == 0) part[tid >> 6] = ssq;
        __syncthreads();
        ssq = 0.f;
#pragma unroll
        for (int i = 0; i < T / 64; i++) ssq += part[i];
    }
    const float inv = 1.0f / sqrtf(ssq / (float)a.cols + a.eps);
    auto put = [&](uint32_t col, const float (&v)[8], const float (&w)[8]) {   // (all 16 lanes of a block that has any column)
        float y[8] = {};
        const bool in = col < a.cols;
        if (in && a.sum) norm_store8<DT, PAST>(a.sum, at + col, v);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = v[j] * w[j] * inv;
        const float scale = fp8_scale(seg16_max(fp8_most(y)));
        if (in) {
            const uint2 codes = fp8_codes(y, scale);
            norm_put<2, PAST>(a.codes + at + col, {codes.x, codes.y});
        }
        if (in && col % kFp8Block == 0) a.scales[(size_t)row * blocks + col / kFp8Block] = scale;
    };
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = (i * T + tid) * 8;
            if constexpr (!AHEAD)
                if (col < a.cols) fp8_load8<DT>(a.weight, col, weights[0]);
            put(col, h[i], weights[AHEAD ? i : 0]);
        }
    } else {
        for (uint32_t col = tid * 8; col / kFp8Block < blocks; col += T * 8) {
            float v[8] = {}, w[8] = {};
            if (col < a.cols) {
                sum8(col, v);
                fp8_load8<DT>(a.weight, col, w);
            }
            put(col, v, w);
        }
    }
}

template <int T, int V> int launch(int dtype, const NormFp8Args& p, const LaunchCtx& lc) {
    NormFp8Args a = p;
    const void* fn[2][3] = {{(const void*)norm_fp8_kernel<DT_F32, T, V, false>, (const void*)norm_fp8_kernel<DT_F16, T, V, false>, (const void*)norm_fp8_kernel<DT_BF16, T, V, false>},
                            {(const void*)norm_fp8_kernel<DT_F32, T, V, true>, (const void*)norm_fp8_kernel<DT_F16, T, V, true>, (const void*)norm_fp8_kernel<DT_BF16, T, V, true>}};
    constexpr uint32_t rows = T < 256 ? 256 / T : 1, threads = T < 256 ? 256 : T;
    const uint64_t groups = ((uint64_t)a.rows + rows - 1) / rows;
    if (groups > max_workgroups(threads)) return fail(ERR_SHAPE, "more rows than a launch can have workgroups");
    void* args[] = {&a};
    MTQ_HIP(launch_kernel(fn[(uint64_t)a.rows * a.cols >= kLarge][dtype], dim3((uint32_t)groups), dim3(threads), args, 0, lc));
    return ERR_OK;
}

}  // namespace

int launch_norm_fp8(int dtype, const NormFp8Args& p, const LaunchCtx& lc) {
    // A wave a row while two vectors a lane hold it, then workgroups of 256 to 1024 threads: fewer vectors a thread are a shorter way for a few rows, and more
    // threads without any work a loss for many (8192 x 2048 bf16: 23.3 us with 256 threads, 26.1 with 512; 2048 x 8192: 20.8 with 512, 21.6 with 256).
    if (p.cols <= 1024) return launch<64, 2>(dtype, p, lc);
    if (p.cols <= 2048) return launch<256, 1>(dtype, p, lc);
    if (p.cols <= 8192) return launch<512, 2>(dtype, p, lc);
    if (p.cols <= 16384) return launch<1024, 2>(dtype, p, lc);
    if (p.cols <= 65536) return launch<1024, 8>(dtype, p, lc);
    return launch<1024, 0>(dtype, p, lc);
}

}  // namespace mtq
