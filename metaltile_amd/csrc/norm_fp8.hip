// Residual addition, RMS norm and quantising into 8-bit floating point (fp8_common.h), in one read of the rows and one write of the sums and codes.
//   h = x + r,  y = (h w) / sqrt(sum h^2 / cols + eps),  a scale and codes of y for each 128 of a row
// Bound by memory; the rows of a decode step by latency. A row stays in registers between its sum of squares and its codes, eight elements a lane
// and 16 lanes a block of 128, as in the quantiser. Rows of more than 65536 elements are read again.
#include "fp8_common.h"

namespace mtq {

namespace {

template <int DT> __device__ __forceinline__ void norm_store8(void* p, size_t i, const float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t)f32_to_elem_bits<DT>(v[2 * j]) | (uint32_t)f32_to_elem_bits<DT>(v[2 * j + 1]) << 16;
        *(uint4*)((uint16_t*)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// T threads a row, V vectors of eight a thread held in registers; V 0: any length, read twice. Workgroups of max(T, 256) threads.
template <int DT, int T, int V> __global__ __launch_bounds__(T < 256 ? 256 : T) void norm_fp8_kernel(NormFp8Args a) {
    constexpr int ROWS = T < 256 ? 256 / T : 1, HELD = V ? V : 1;
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
    float h[HELD][8] = {}, ssq = 0.f;
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = (i * T + tid) * 8;
            if (col < a.cols) sum8(col, h[i]);
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
    auto put = [&](uint32_t col, const float (&v)[8]) {   // (all 16 lanes of a block that has any column)
        float y[8] = {};
        const bool in = col < a.cols;
        if (in) {
            fp8_load8<DT>(a.weight, col, y);
            if (a.sum) norm_store8<DT>(a.sum, at + col, v);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = v[j] * y[j] * inv;
        const float scale = fp8_scale(seg16_max(fp8_most(y)));
        if (in) *(uint2*)(a.codes + at + col) = fp8_codes(y, scale);
        if (in && col % kFp8Block == 0) a.scales[(size_t)row * blocks + col / kFp8Block] = scale;
    };
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; i++) put((i * T + tid) * 8, h[i]);
    } else {
        for (uint32_t col = tid * 8; col / kFp8Block < blocks; col += T * 8) {
            float v[8] = {};
            if (col < a.cols) sum8(col, v);
            put(col, v);
        }
    }
}

template <int T, int V> int launch(int dtype, const NormFp8Args& p, const LaunchCtx& lc) {
    NormFp8Args a = p;
    const void* fn[] = {(const void*)norm_fp8_kernel<DT_F32, T, V>, (const void*)norm_fp8_kernel<DT_F16, T, V>, (const void*)norm_fp8_kernel<DT_BF16, T, V>};
    constexpr uint32_t rows = T < 256 ? 256 / T : 1, threads = T < 256 ? 256 : T;
    const uint64_t groups = ((uint64_t)a.rows + rows - 1) / rows;
    if (groups > max_workgroups(threads)) return fail(ERR_SHAPE, "more rows than a launch can have workgroups");
    void* args[] = {&a};
    MTQ_HIP(launch_kernel(fn[dtype], dim3((uint32_t)groups), dim3(threads), args, 0, lc));
    return ERR_OK;
}

}  // namespace

int launch_norm_fp8(int dtype, const NormFp8Args& p, const LaunchCtx& lc) {
    if (p.cols <= 1024) return launch<64, 2>(dtype, p, lc);
    if (p.cols <= 8192) return launch<256, 4>(dtype, p, lc);
    if (p.cols <= 65536) return launch<1024, 8>(dtype, p, lc);
    return launch<1024, 0>(dtype, p, lc);
}

}  // namespace mtq
