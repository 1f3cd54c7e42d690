// Quantising into 8-bit floating point with a scale for each block of 128 (fp8_common.h): one read of the elements, one write of the codes.
// Bound by memory: a block stays in registers between its maximum and its codes.
#include "fp8_common.h"

namespace mtq {

namespace {

struct Fp8QuantArgs {
    const void* x;
    uint8_t* codes;
    float* scales;
    uint32_t rows, cols, blocks;   // blocks: ceil(cols / 128)
};

// 1 x 128 blocks, one to 16 lanes of eight elements each.
template <int DT> __global__ __launch_bounds__(256) void fp8_quantize_rows_kernel(Fp8QuantArgs a) {
    // The workgroup's first block by one division for all lanes, a lane's from there (blocks are less than 2^23).
    const uint64_t at0 = (uint64_t)blockIdx.x * 16, at = at0 + (threadIdx.x >> 4);
    if (at >= (uint64_t)a.rows * a.blocks) return;   // (all 16 lanes of a block or none)
    const uint32_t row0 = at0 <= UINT32_MAX ? (uint32_t)at0 / a.blocks : (uint32_t)(at0 / a.blocks), from = (uint32_t)(at0 - (uint64_t)row0 * a.blocks) + (threadIdx.x >> 4);
    const uint32_t on = from / a.blocks, row = row0 + on, block = from - on * a.blocks, col = block * kFp8Block + (threadIdx.x & 15u) * 8;
    const bool in = col < a.cols;
    const size_t i = (size_t)row * a.cols + col;
    float v[8] = {};
    if (in) fp8_load8<DT>(a.x, i, v);
    const float scale = fp8_scale(seg16_max(fp8_most(v)));
    if (in) *(uint2*)(a.codes + i) = fp8_codes(v, scale);
    if ((threadIdx.x & 15u) == 0) a.scales[at] = scale;
}

// 128 x 128 blocks, one to a workgroup: 16 lanes along a row, 16 rows at a time. Where rows are not whole lines, neighbours share lines of both
// and go to one XCD (14300 x 4144 bf16: 47.7 -> 39.8 us); else in turn (8192 x 8192 f32: 60.7 us against 64.1 in runs).
template <int DT> __global__ __launch_bounds__(256) void fp8_quantize_tiles_kernel(Fp8QuantArgs a) {
    __shared__ float part[4];
    const uint32_t unit = a.cols % 128 ? xcd_run(blockIdx.x, gridDim.x) : blockIdx.x, block = unit % a.blocks, rb = unit / a.blocks;
    const uint32_t col = block * kFp8Block + (threadIdx.x & 15u) * 8, row0 = rb * kFp8Block + (threadIdx.x >> 4);
    const bool in = col < a.cols;
    float v[8][8] = {}, most = 0.f;
#pragma unroll
    for (int p = 0; p < 8; p++)
        if (in && row0 + 16 * p < a.rows) fp8_load8<DT>(a.x, (size_t)(row0 + 16 * p) * a.cols + col, v[p]);
#pragma unroll
    for (int p = 0; p < 8; p++) most = fmaxf(most, fp8_most(v[p]));
    most = seg16_max(most);
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64));
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    const float scale = fp8_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
#pragma unroll
    for (int p = 0; p < 8; p++)
        if (in && row0 + 16 * p < a.rows) *(uint2*)(a.codes + (size_t)(row0 + 16 * p) * a.cols + col) = fp8_codes(v[p], scale);
    if (threadIdx.x == 0) a.scales[unit] = scale;
}

}  // namespace

int launch_fp8_quantize(int dtype, const void* x, void* codes, float* scales, uint32_t rows, uint32_t cols, uint32_t block_rows, const LaunchCtx& lc) {
    Fp8QuantArgs a{x, (uint8_t*)codes, scales, rows, cols, (cols + kFp8Block - 1) / kFp8Block};
    const bool tiles = block_rows > 1;
    const uint64_t units = tiles ? (uint64_t)((rows + kFp8Block - 1) / kFp8Block) * a.blocks : ((uint64_t)rows * a.blocks + 15) / 16;
    if (units > max_workgroups(256)) return fail(ERR_SHAPE, "more blocks than a launch can have workgroups");
    const void* rows_fn[] = {(const void*)fp8_quantize_rows_kernel<DT_F32>, (const void*)fp8_quantize_rows_kernel<DT_F16>, (const void*)fp8_quantize_rows_kernel<DT_BF16>};
    const void* tiles_fn[] = {(const void*)fp8_quantize_tiles_kernel<DT_F32>, (const void*)fp8_quantize_tiles_kernel<DT_F16>, (const void*)fp8_quantize_tiles_kernel<DT_BF16>};
    void* args[] = {&a};
    MTQ_HIP(launch_kernel((tiles ? tiles_fn : rows_fn)[dtype], dim3((uint32_t)units), dim3(256), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
