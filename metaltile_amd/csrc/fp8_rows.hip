// Few activation rows times a weight matrix in 8-bit floating point (fp8_common.h): bound by the one read of the weights.
//
//   out[m, n] = sum over blocks b of xs[m, b] ws[n / 128, b] (sum over b's k of x[m, k] w[n, k])
//
// The inner sum is one 16 x 16 x 128 matrix instruction; its two scales differ by block and by row of the result, so they are multiplied
// in behind it, one f32 FMA a value. A workgroup has 16 NT weight rows and 16 MT activation rows, and its waves share the blocks of K; the
// weights go from memory to the matrix cores' registers, the next blocks' while those at hand are multiplied, and the waves' sums meet in
// LDS. The weights are the instruction's rows, so that a lane has four neighbouring n of one m, and one scale for all of them.
// A few rows can come as they are: the workgroup quantises them into LDS while its first weights are on their way.
#include "fp8_common.h"

namespace mtq {

namespace {

template <int DT, int MT, int NT, int NW, bool FUSED> __global__ __launch_bounds__(64 * NW) void fp8_rows_kernel(Fp8Args a) {
    static_assert(!FUSED || MT == 1, "");
    constexpr int D = MT == 1 ? 4 / NT : 2;   // a wave's blocks at a time
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // sums [NW][NT][MT][64]; before them the quantised rows and their scales
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const uint32_t r = lane & 15u, g = lane >> 4, blocks = fp8_blocks(a.K);
    const uint8_t* w[NT];
    const float* ws[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint32_t n = n0 + 16 * t + r, nb = (n0 + 16 * t < a.N ? n0 + 16 * t : a.N - 1) / kFp8Block;
        w[t] = a.w + (size_t)(n < a.N ? n : a.N - 1) * a.K + 16 * g;
        ws[t] = a.ws + (size_t)nb * blocks;
    }
    // Pieces g and 4 + g of block b of a row; a piece behind the row's end is zeros.
    auto piece = [&](const uint8_t* row, uint32_t b, int h) {
        const uint32_t k = b * kFp8Block + 64 * h;
        if ((b + 1) * kFp8Block <= a.K) return *(const uint4*)(row + k);
        return k + 16 * g < a.K ? *(const uint4*)(row + k) : make_uint4(0, 0, 0, 0);
    };
    uint4 wv[2][D][NT][2];
    auto load = [&](int to, uint32_t b0) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const uint32_t b = b0 + d * NW;
            if (b < blocks)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int h = 0; h < 2; h++) wv[to][d][t][h] = piece(w[t], b, h);
        }
    };
    const uint8_t* x[MT];
    const float* xs[MT];
    const uint32_t pitch = blocks * kFp8Block + 16;   // of a quantised row in LDS (rows begin in different banks)
    float* lds_scales = (float*)(lds + (size_t)a.M * pitch);
    load(0, wave);
    if constexpr (FUSED) {
        for (uint32_t u = threadIdx.x >> 4; u < a.M * blocks; u += 4 * NW) {
            const uint32_t row = u / blocks, b = u % blocks, k = b * kFp8Block + (lane & 15u) * 8;
            float v[8] = {};
            if (k < a.K) fp8_load8<DT>(a.x, (size_t)row * a.K + k, v);
            const float scale = fp8_scale(seg16_max(fp8_most(v)));
            *(uint2*)(lds + (size_t)row * pitch + k) = fp8_codes(v, scale);
            if ((lane & 15u) == 0) lds_scales[u] = scale;
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const uint32_t m = m0 + 16 * t + r, row = m < a.M ? m : a.M - 1;
            x[t] = (const uint8_t*)a.x + (size_t)row * a.K + 16 * g;
            xs[t] = a.xs + (size_t)row * blocks;
        }
    }
    const uint32_t mine = r < a.M ? r : a.M - 1;   // (FUSED: a row past the last reads the last's, and its results are not stored)
    fp8_f32x4 acc[MT][NT] = {};
    auto multiply = [&](int from, uint32_t b0) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const uint32_t b = b0 + d * NW;
            if (b >= blocks) break;
            float sw[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) sw[t] = ws[t][b];
            uint4 xv[MT][2];
            float sx[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) {
                if constexpr (FUSED) {
                    const uint8_t* p = lds + (size_t)mine * pitch + b * kFp8Block + 16 * g;
                    xv[t][0] = *(const uint4*)p;
                    xv[t][1] = *(const uint4*)(p + 64);
                    sx[t] = lds_scales[mine * blocks + b];
                } else {
                    xv[t][0] = piece(x[t], b, 0);
                    xv[t][1] = piece(x[t], b, 1);
                    sx[t] = xs[t][b];
                }
            }
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    const fp8_f32x4 p = fp8_mfma<DT>(wv[from][d][u][0], wv[from][d][u][1], xv[t][0], xv[t][1]);
                    const float s = sx[t] * sw[u];
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[t][u][i] = fmaf(p[i], s, acc[t][u][i]);
                }
        }
    };
    for (uint32_t b0 = wave; b0 < blocks; b0 += 2 * NW * D) {
        load(1, b0 + NW * D);
        multiply(0, b0);
        load(0, b0 + 2 * NW * D);
        multiply(1, b0 + NW * D);
    }
    if constexpr (FUSED) __syncthreads();   // (the quantised rows are no longer read)
    fp8_f32x4* part = (fp8_f32x4*)lds;
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int u = 0; u < NT; u++) part[((wave * MT + t) * NT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
    for (uint32_t j = wave; j < MT * NT; j += NW) {
        fp8_f32x4 sum = part[j * 64 + lane];
        for (int v = 1; v < NW; v++) sum += part[(v * MT * NT + j) * 64 + lane];
        const uint32_t m = m0 + 16 * (j / NT) + r, n = n0 + 16 * (j % NT) + 4 * g;
        if (m < a.M) fp8_store4<DT>(a.out, m, n, a.N, sum);
    }
}

template <int DT> const void* rows_fn(int mt, int nw) {
    if (mt == 1) return nw == 16 ? (const void*)fp8_rows_kernel<DT, 1, 1, 16, false> : nw == 8 ? (const void*)fp8_rows_kernel<DT, 1, 1, 8, false> : (const void*)fp8_rows_kernel<DT, 1, 1, 4, false>;
    return mt == 2 ? (const void*)fp8_rows_kernel<DT, 2, 2, 8, false> : (const void*)fp8_rows_kernel<DT, 4, 2, 4, false>;
}
template <int DT> const void* fused_fn(int nw) {
    return nw == 16 ? (const void*)fp8_rows_kernel<DT, 1, 1, 16, true> : nw == 8 ? (const void*)fp8_rows_kernel<DT, 1, 1, 8, true> : (const void*)fp8_rows_kernel<DT, 1, 1, 4, true>;
}
// Waves that share the blocks of 16 weight rows: four where that makes 2048 of them or more, else up to sixteen.
int waves_of(const Fp8Args& a) {
    const uint64_t groups = (uint64_t)((a.N + 15) / 16) * ((a.M + 15) / 16);
    const uint32_t blocks = fp8_blocks(a.K);
    int nw = 4;
    while (nw < 16 && groups * nw < 2048 && (uint32_t)nw < blocks) nw *= 2;
    return nw;
}
size_t fused_lds(const Fp8Args& a, int nw) {
    const size_t blocks = fp8_blocks(a.K), rows = a.M * (blocks * kFp8Block + 16) + a.M * blocks * 4, sums = (size_t)nw * 1024;
    return rows > sums ? rows : sums;
}

}  // namespace

// A workgroup's time is that of bringing its rows, of x and of w, through its CU's first-level cache, so the rows of x are spread over as many
// workgroups as there are CUs, the weights read again from the L2, and each takes more of them only where there would be more workgroups than
// that (bf16, K = 4096, us with 16 / 32 / 64 rows of x a workgroup and in tiles: 64 x 1024 10.5 / 13.6 / 19.0 / 23.9; 64 x 4096 23.0 / 14.3 /
// 19.8 / 24.4; 128 x 4096 40.6 / 23.3 / 20.5 / 26.0; 33 x 14336 47.6 / 33.2 / 27.1 / 24.0). f32 results, twice the time in tiles, go there behind
// two workgroups a CU (256 x 4096: 35.7 against 42.8). Tiles have 31-bit offsets in their rows.
int fp8_rows_tiles(int dtype, const Fp8Args& a) {
    const uint64_t cus = (uint64_t)fp8_num_cus();
    auto groups = [&](uint32_t mt, uint32_t nt) { return (uint64_t)((a.M + 16 * mt - 1) / (16 * mt)) * ((a.N + 16 * nt - 1) / (16 * nt)); };
    if (a.M <= 16 || groups(1, 1) <= cus) return 1;
    if (a.M <= 32 || groups(2, 2) <= cus) return 2;
    return groups(4, 2) <= (dtype == DT_F32 ? 2 : 1) * cus || a.K > kFp8TilesLongest ? 4 : 0;
}

// A workgroup's rows of x are sixteen at most, and all of K has to be in LDS.
bool fp8_fused_fits(const Fp8Args& p) { return p.M <= 16 && fused_lds(p, 16) <= 160 * 1024; }
// Every workgroup quantises the rows anew, which costs less than a launch of its own (3 us) for one row, or for a few where the workgroups are
// few too (us, fused and not, K = 4096: 1 x 14336 16.9 / 18.2; 4 x 1024 6.8 / 9.0; 2 x 14336 19.4 / 18.6; 4 x 14336 24.5 / 19.7).
bool fp8_fused_takes(const Fp8Args& p) { return (p.M == 1 || (p.M <= 4 && (uint64_t)p.M * ((p.N + 15) / 16) <= 256)) && fused_lds(p, 16) <= 40 * 1024; }

int launch_fp8_fused(int dtype, const Fp8Args& p, const LaunchCtx& lc) {
    Fp8Args a = p;
    const int nw = waves_of(a);
    const void* fn = dtype == DT_F32 ? fused_fn<DT_F32>(nw) : dtype == DT_F16 ? fused_fn<DT_F16>(nw) : fused_fn<DT_BF16>(nw);
    const size_t lds = fused_lds(a, nw);
    void* args[] = {&a};
    MTQ_HIP(set_max_dynamic_lds(fn, lds));
    MTQ_HIP(launch_kernel(fn, dim3((a.N + 15) / 16), dim3(64 * nw), args, lds, lc));
    return ERR_OK;
}

static dim3 rows_grid(const Fp8Args& a, int mt, int& nt, int& nw) {
    nt = mt == 1 ? 1 : 2;
    nw = mt == 1 ? waves_of(a) : mt == 2 ? 8 : 4;
    return dim3((a.N + 16 * nt - 1) / (16 * nt), (a.M + 16 * mt - 1) / (16 * mt));
}
bool fp8_rows_fit(const Fp8Args& a, int mt) {
    int nt, nw;
    const dim3 grid = rows_grid(a, mt, nt, nw);
    return grid.x <= max_workgroups(64 * nw) && grid.y <= 65535u;
}

int launch_fp8_rows(int dtype, const Fp8Args& p, int mt, const LaunchCtx& lc) {
    Fp8Args a = p;
    int nt, nw;
    const dim3 grid = rows_grid(a, mt, nt, nw);
    const void* fn = dtype == DT_F32 ? rows_fn<DT_F32>(mt, nw) : dtype == DT_F16 ? rows_fn<DT_F16>(mt, nw) : rows_fn<DT_BF16>(mt, nw);
    const size_t lds = (size_t)nw * nt * mt * 1024;
    void* args[] = {&a};
    MTQ_HIP(set_max_dynamic_lds(fn, lds));
    MTQ_HIP(launch_kernel(fn, grid, dim3(64 * nw), args, lds, lc));
    return ERR_OK;
}

}  // namespace mtq
