// Many activation rows times a weight matrix in 8-bit floating point (fp8_common.h): bound by the matrix cores.
//
//   out[m, n] = sum over blocks b of xs[m, b] ws[n / 128, b] (sum over b's k of x[m, k] w[n, k])
//
// A workgroup has a tile of BM x BN results, its waves WM x WN parts of it in registers. K goes by in blocks of 128: both operands' codes
// come into LDS by load-to-LDS instructions while the block before is computed (two stages), 16 bytes a lane, and the 16-byte pieces of a row
// are kept in an order turned by the row's number (piece c of row r lies at c ^ (r & 7)), so that the sixteen rows that a matrix
// instruction reads at once lie in different banks. A block's sums come out of one matrix instruction from zero, and the two scales are
// multiplied in behind it, one f32 FMA a value, which the vector units do beside the matrix cores. The weights are the instruction's
// rows: a lane then has four neighbouring n of one m, one scale for all of them.
#include "fp8_common.h"

namespace mtq {

namespace {

// 16 bytes a lane from rsrc + voff (past the end: zeros) to LDS: lane l's at lds + 16 l. No register is written; counts in vmcnt.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // M0 is a reserved register: naming it as clobbered is the point
__device__ __forceinline__ void lds_load16(uint32_t lds, uint32_t voff, __attribute__((ext_vector_type(4))) uint32_t rsrc) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ __attribute__((ext_vector_type(4))) uint32_t tile_rsrc(const uint8_t* base, uint32_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    __attribute__((ext_vector_type(4))) uint32_t r;
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000;
    return r;
}

constexpr uint32_t kOutOfRange = 0x80000000u;   // (a tile's rows are less than 2 GiB)

template <int DT, int BM, int BN, int WM, int WN> __global__ __launch_bounds__(64 * WM * WN) void fp8_tiles_kernel(Fp8Args a, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, STAGE = (BM + BN) * 128, QX = BM / 8 / NW, QW = BN / 8 / NW;
    static_assert(64 * NW >= BM, "a thread brings the scale of a row");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    float* sxs = (float*)(lds + 2 * STAGE);   // [2][64 NW]: of the tile's BM rows (and some behind them)
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15u, g = lane >> 4, wm = wave / WN, wn = wave % WN;
    const uint32_t blocks = (a.K + kFp8Block - 1) / kFp8Block;
    // Workgroups go to the eight XCDs in turn. Each XCD gets a run of neighbouring tiles, in bands of four tiles of n, so that those it has at a
    // time (32) share eight tiles of m and four of n in its L2.
    const uint32_t total = tiles_m * tiles_n, per = total / 8, extra = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    const uint32_t tile = xcd * per + (xcd < extra ? xcd : extra) + at;
    const uint32_t band = tile / (4 * tiles_m), wide = tiles_n - 4 * band < 4 ? tiles_n - 4 * band : 4, in_band = tile - band * 4 * tiles_m;
    const uint32_t m0 = in_band / wide * BM, n0 = (band * 4 + in_band % wide) * BN;
    const uint32_t rows_m = a.M - m0 < BM ? a.M - m0 : BM, rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    const auto rx = tile_rsrc((const uint8_t*)a.x + (size_t)m0 * a.K, rows_m * a.K), rw = tile_rsrc(a.w + (size_t)n0 * a.K, rows_n * a.K);
    const uint32_t chunk = (lane & 7u) ^ (lane >> 3), k_left = a.K - 16 * chunk;   // this lane's piece of a row; the k where it ends being there
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t v0 = (lane >> 3) * a.K + 16 * chunk;
    auto load = [&](uint32_t b, uint32_t stage) {
        const bool in = b * kFp8Block < k_left && 16 * chunk < a.K;
        const uint32_t to = lds0 + stage * STAGE;
        uint32_t v = v0 + b * kFp8Block;
        asm volatile("" : "+v"(v));   // (the pieces' offsets are not kept from block to block: the registers are the results')
#pragma unroll
        for (int q = 0; q < QX; q++) lds_load16(__builtin_amdgcn_readfirstlane(to + (wave * QX + q) * 1024), in ? v + 8 * (wave * QX + q) * a.K : kOutOfRange, rx);
#pragma unroll
        for (int q = 0; q < QW; q++) lds_load16(__builtin_amdgcn_readfirstlane(to + BM * 128 + (wave * QW + q) * 1024), in ? v + 8 * (wave * QW + q) * a.K : kOutOfRange, rw);
    };
    const uint32_t srow = m0 + threadIdx.x < a.M ? m0 + threadIdx.x : a.M - 1;
    const float* sx = a.xs + (size_t)srow * blocks;
    // (a wave's n lie in one block of 128: BN / WN divides it)
    const uint32_t nb = (n0 + wn * (BN / WN)) / kFp8Block, nbs = (a.N + kFp8Block - 1) / kFp8Block;
    const float* sw = a.ws + (size_t)(nb < nbs ? nb : nbs - 1) * blocks;
    fp8_f32x4 acc[TM][TN] = {};
    load(0, 0);
    sxs[threadIdx.x] = sx[0];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint32_t o0 = r * 128 + ((g ^ (r & 7u)) << 4), o1 = o0 ^ 64u;   // pieces g and 4 + g of row r
    for (uint32_t b = 0; b < blocks; b++) {
        const uint32_t s = b & 1u;
        // (no branch in the loop: the compiler would move the scaling below it; behind the last block the loads bring zeros)
        load(b + 1, s ^ 1u);
        const float next = sx[b + 1 < blocks ? b + 1 : b];
        const float w = sw[b];
        const uint32_t xt = s * STAGE + wm * (BM / WM) * 128, wt = s * STAGE + BM * 128 + wn * (BN / WN) * 128;
        uint4 wv[TN][2];
#pragma unroll
        for (int j = 0; j < TN; j++) {
            wv[j][0] = *(const uint4*)(lds + wt + j * 2048 + o0);
            wv[j][1] = *(const uint4*)(lds + wt + j * 2048 + o1);
        }
        // The next piece of x is read, and the last sums are scaled, while the matrix cores have this piece.
        uint4 xv[2][2];
        float scale[2] = {};
        fp8_f32x4 p[2][TN];
        auto read = [&](int t) {
            xv[t & 1][0] = *(const uint4*)(lds + xt + t * 2048 + o0);
            xv[t & 1][1] = *(const uint4*)(lds + xt + t * 2048 + o1);
            scale[t & 1] = sxs[s * 64 * NW + wm * (BM / WM) + 16 * t + r] * w;
        };
        auto add = [&](int t, float by) {
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t][j][i] = fmaf(p[t & 1][j][i], by, acc[t][j][i]);
        };
        read(0);
        float before = 0.f;
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const uint4 x0 = xv[t & 1][0], x1 = xv[t & 1][1];
            const float now = scale[t & 1];
            if (t + 1 < TM) read(t + 1);
#pragma unroll
            for (int j = 0; j < TN; j++) p[t & 1][j] = fp8_mfma<DT>(wv[j][0], wv[j][1], x0, x1);
            if (t) add(t - 1, before);
            before = now;
            __builtin_amdgcn_sched_barrier(0);
        }
        add(TM - 1, before);
        sxs[(s ^ 1u) * 64 * NW + threadIdx.x] = next;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const bool whole = (a.N * ES) % (4 * ES) == 0 && (uintptr_t)a.out % (4 * ES) == 0;
#pragma unroll
    for (int t = 0; t < TM; t++) {
        const uint32_t m = m0 + wm * (BM / WM) + 16 * t + r;
        if (m >= a.M) continue;
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const uint32_t n = n0 + wn * (BN / WN) + 16 * j + 4 * g;
            const size_t i0 = (size_t)m * a.N + n;
            if (whole && n < a.N) {
                if constexpr (DT == DT_F32) {
                    *(fp8_f32x4*)((float*)a.out + i0) = acc[t][j];
                } else {
                    *(uint2*)((uint16_t*)a.out + i0) = make_uint2(f32_to_elem_bits<DT>(acc[t][j][0]) | (uint32_t)f32_to_elem_bits<DT>(acc[t][j][1]) << 16,
                                                                  f32_to_elem_bits<DT>(acc[t][j][2]) | (uint32_t)f32_to_elem_bits<DT>(acc[t][j][3]) << 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (n + i < a.N) store_elem<DT>(a.out, i0 + i, acc[t][j][i]);
            }
        }
    }
}

template <int BM, int BN, int WM, int WN, int... DTS> int launch(int dtype, const Fp8Args& p, const LaunchCtx& lc) {
    Fp8Args a = p;
    uint32_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    if ((uint64_t)tm * tn > 0x7FFFFFFFull) return fail(ERR_SHAPE, "more tiles than a launch can have workgroups");
    const void* fn = nullptr;
    ((dtype == DTS ? (void)(fn = (const void*)fp8_tiles_kernel<DTS, BM, BN, WM, WN>) : (void)0), ...);
    constexpr size_t lds = 2 * (BM + BN) * 128 + 2 * 64 * WM * WN * sizeof(float);
    MTQ_HIP(set_max_dynamic_lds(fn, lds));
    void* args[] = {&a, &tm, &tn};
    MTQ_HIP(launch_kernel(fn, dim3(tm * tn), dim3(64 * WM * WN), args, lds, lc));
    return ERR_OK;
}

}  // namespace

bool fp8_tiles_takes(int dtype, const Fp8Args& p) { return p.M > 64 && p.K <= (1u << 22); }   // (a tile's rows have 31-bit offsets)

int launch_fp8_tiles(int dtype, const Fp8Args& p, const LaunchCtx& lc) {
    const uint64_t large = (uint64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
    if (dtype != DT_F32 && large >= 200) return launch<256, 256, 2, 4, DT_F16, DT_BF16>(dtype, p, lc);
    return launch<128, 128, 2, 2, DT_F32, DT_F16, DT_BF16>(dtype, p, lc);
}

}  // namespace mtq
