// Many activation rows times a weight matrix in 8-bit floating point (fp8_common.h): bound by the matrix cores.
//
//   out[m, n] = sum over blocks b of xs[m, b] ws[n / 128, b] (sum over b's k of x[m, k] w[n, k])
//
// A workgroup has a tile of BM x BN results, its waves WM x WN parts of it in registers. K goes by in blocks of 128: both operands' codes
// come into LDS by load-to-LDS instructions, 16 bytes a lane, while the blocks before are computed (in two or four stages), and the 16-byte
// pieces of a row are kept in an order turned by the row's number (piece c of row r lies at c ^ (r & 7)), so that the sixteen rows that a
// matrix instruction reads at once lie in different banks. A block's sums come out of one matrix instruction from zero, and the two scales
// are multiplied in behind it, one f32 FMA a value, which the vector units do beside the matrix cores. The weights are the instruction's
// rows: a lane then has four neighbouring n of one m, one scale for all of them.
//
// The waves meet once a block, before its last step rather than behind it: all of the block is in registers then, so its stage is free, and
// the next block's first operands are read while the last step's products and sums are computed (8 waves of 128 x 64 each, 4096 rows x 14336
// x 4096 with the quantising: 324 -> 265 us). The next loads are issued a quarter at each of four steps, as eight at once keep the LDS from
// the reads (265 -> 247 us).
//
// 256 x 256 tiles do twice the products of 128 x 128 ones for each byte that they read, but come in few: 224 of them (1024 x 14336) take as
// long as 256, and what is left over after whole rounds costs a round. Their time by the round, with K = 4096: 58 us, as tiles cut in two 38,
// of 128 x 128 ones 25 (16 waves, four stages). Where 128 x 64 ones (8 waves) are no more than the CUs they end sooner: 128 x 14336 23.4 us with
// the quantising against 26.8, 512 x 4096 23.6 against 26.5. f32 results, whose codes are unpacked to bf16 for the products (fp8_common.h), have two
// workgroups of 128 x 128 a CU (4096^3: 143 us against 231 with one and four stages).
#include "fp8_common.h"

namespace mtq {

namespace {

// 16 bytes a lane from rsrc + voff (past the end: zeros) to LDS: lane l's at lds + 16 l. No register is written; counts in vmcnt. M0 is read one wait
// state behind its write at the earliest, which no one but this block sees to.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // M0 is a reserved register: naming it as clobbered is the point
__device__ __forceinline__ void lds_load16(uint32_t lds, uint32_t voff, __attribute__((ext_vector_type(4))) uint32_t rsrc) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
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
constexpr uint32_t kWindow = 4;                 // blocks whose scales of x are brought in together, 16 bytes a row

// The tile of BM x BN results at (m0, n0), which is one with a row in it.
template <int DT, int BM, int BN, int WM, int WN, int STAGES> __device__ __forceinline__ void fp8_tile(const Fp8Args& a, uint32_t m0, uint32_t n0, uint8_t* lds) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, STAGE = (BM + BN) * 128, QX = BM / 8 / NW, QW = BN / 8 / NW;
    static_assert(64 * NW >= BM && (STAGES & (STAGES - 1)) == 0, "a lane brings the scales of a row; stages are counted by their low bits");
    constexpr uint32_t SCALES = STAGES * STAGE;   // behind the stages: [2][BM][kWindow] scales of x
    constexpr int PARTS = TM > 4 ? 4 : TM > 2 ? 2 : 1;   // in which a block's loads are issued, one at each of as many steps
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15u, g = lane >> 4, wm = wave / WN, wn = wave % WN;
    const uint32_t blocks = fp8_blocks(a.K);
    const uint32_t rows_m = a.M - m0 < BM ? a.M - m0 : BM, rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    const auto rx = tile_rsrc((const uint8_t*)a.x + (size_t)m0 * a.K, rows_m * a.K), rw = tile_rsrc(a.w + (size_t)n0 * a.K, rows_n * a.K);
    const auto rs = tile_rsrc((const uint8_t*)(a.xs + (size_t)m0 * blocks), rows_m * blocks * 4);
    const uint32_t chunk = (lane & 7u) ^ (lane >> 3), k_left = a.K - 16 * chunk;   // this lane's piece of a row; the k where it ends being there
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t v0 = (lane >> 3) * a.K + 16 * chunk;
    auto load = [&](uint32_t b, int from, int end) {   // a part of block b's codes into its stage; behind the last block: zeros
        const bool in = b * kFp8Block < k_left && 16 * chunk < a.K;
        const uint32_t to = lds0 + (b & (STAGES - 1)) * STAGE;
        uint32_t v = in ? v0 + b * kFp8Block : kOutOfRange;   // (rows are added here and not as a scalar offset: some are behind the tile's last)
        asm volatile("" : "+v"(v));                           // (the pieces' offsets are not kept from block to block: the registers are the results')
#pragma unroll
        for (int q = 0; q < QX; q++) if (q >= from && q < end) lds_load16(__builtin_amdgcn_readfirstlane(to + (wave * QX + q) * 1024), v + 8 * (wave * QX + q) * a.K, rx);
#pragma unroll
        for (int q = 0; q < QW; q++) if (QX + q >= from && QX + q < end) lds_load16(__builtin_amdgcn_readfirstlane(to + BM * 128 + (wave * QW + q) * 1024), v + 8 * (wave * QW + q) * a.K, rw);
    };
    auto load_scales = [&](uint32_t w) {   // window w's, of row 64 wave + lane (what is behind a row's last block is not used)
        if (wave >= BM / 64) return;
        const uint32_t row = 64 * wave + lane;
        lds_load16(__builtin_amdgcn_readfirstlane(lds0 + SCALES + (w & 1u) * (BM * kWindow * 4) + wave * 1024), row < rows_m ? (row * blocks + w * kWindow) * 4 : kOutOfRange, rs);
    };
    // (a wave's n lie in one block of 128: BN / WN divides it)
    const uint32_t nb = (n0 + wn * (BN / WN)) / kFp8Block, nbs = fp8_blocks(a.N);
    const float* sw = a.ws + (size_t)(nb < nbs ? nb : nbs - 1) * blocks;
    fp8_f32x4 acc[TM][TN] = {};
    load_scales(0);
#pragma unroll
    for (int b = 0; b < STAGES; b++) load(b, 0, QX + QW);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    auto meet = [&] {   // the next block is whole when no more of a wave's loads are on their way than those for the stages behind it, and all waves say so
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * (QX + QW)) : "memory");
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    if (wm * (BM / WM) >= rows_m) {   // all of this wave's rows are behind the last: it has loads only, and leaves the LDS to the others
        static_assert(BM / 64 <= WN, "the scales are brought by waves of the first rows");
        for (uint32_t b = 0; b < blocks; b++) {
            meet();
            load(b + STAGES, 0, QX + QW);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        return;
    }
    const uint32_t o0 = r * 128 + ((g ^ (r & 7u)) << 4), o1 = o0 ^ 64u;   // pieces g and 4 + g of row r
    uint4 wv[TN][2], xv[2][2];
    float scale[2] = {};
    fp8_f32x4 p[2][TN];
    auto read_w = [&](uint32_t b) {
        const uint8_t* wt = lds + (b & (STAGES - 1)) * STAGE + BM * 128 + wn * (BN / WN) * 128;
#pragma unroll
        for (int j = 0; j < TN; j++) {
            wv[j][0] = *(const uint4*)(wt + j * 2048 + o0);
            wv[j][1] = *(const uint4*)(wt + j * 2048 + o1);
        }
    };
    auto read_x = [&](uint32_t b, int t, float w) {
        const uint8_t* xt = lds + (b & (STAGES - 1)) * STAGE + wm * (BM / WM) * 128 + t * 2048;
        xv[t & 1][0] = *(const uint4*)(xt + o0);
        xv[t & 1][1] = *(const uint4*)(xt + o1);
        scale[t & 1] = ((const float*)(lds + SCALES))[((b / kWindow & 1u) * BM + wm * (BM / WM) + 16 * t + r) * kWindow + b % kWindow] * w;
    };
    auto add = [&](int t, float by) {
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[t][j][e] = fmaf(p[t & 1][j][e], by, acc[t][j][e]);
    };
    float w = sw[0];
    read_x(0, 0, w);
    read_w(0);
    for (uint32_t b = 0; b < blocks; b++) {
        const float w_next = sw[b + 1 < blocks ? b + 1 : b];
        if (b % kWindow == 0) load_scales(b / kWindow + 1);
        float before = 0.f;
        // The next piece of x is read, and the last sums are scaled, while the matrix cores have this piece.
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const float now = scale[t & 1];
            if (t + 1 < TM) {
                read_x(b, t + 1, w);
            } else {
                meet();   // (all of this block is read: its stage is free behind this)
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < TN; j++) p[t & 1][j] = fp8_mfma<DT>(wv[j][0], wv[j][1], xv[t & 1][0], xv[t & 1][1]);
            if (t + 1 == TM) {   // (the last pieces of a block are multiplied while the next block's first are read; behind the last block: zeros)
                read_x(b + 1, 0, w_next);
                read_w(b + 1);
                load(b + STAGES, 0, (QX + QW) / PARTS);
            } else if (t + 1 < PARTS && b) {
                load(b + STAGES - 1, (t + 1) * (QX + QW) / PARTS, (t + 2) * (QX + QW) / PARTS);
            }
            if (t) add(t - 1, before);
            before = now;
            __builtin_amdgcn_sched_barrier(0);
        }
        add(TM - 1, before);
        w = w_next;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (nothing is on its way into LDS that another workgroup may have next)
#pragma unroll
    for (int t = 0; t < TM; t++) {
        const uint32_t m = m0 + wm * (BM / WM) + 16 * t + r;
        if (m >= a.M) continue;
#pragma unroll
        for (int j = 0; j < TN; j++) fp8_store4<DT>(a.out, m, n0 + wn * (BN / WN) + 16 * j + 4 * g, a.N, acc[t][j]);
    }
}

// One workgroup a tile for the first `whole` tiles; HALVES: two for each of the others, the upper half of its rows and the lower.
template <int DT, int BM, int BN, int WM, int WN, int STAGES, bool HALVES> __global__ __launch_bounds__(64 * WM * WN) void fp8_tiles_kernel(Fp8Args a, uint32_t tiles_m, uint32_t tiles_n, uint32_t whole) {
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const bool half = HALVES && blockIdx.x >= whole;
    const uint32_t i = half ? xcd_run(blockIdx.x - whole, 2 * (tiles_m * tiles_n - whole)) : xcd_run(blockIdx.x, whole), tile = half ? whole + i / 2 : i;
    // In bands of four tiles of n, so that the tiles that an XCD has at a time (32) share eight tiles of m and four of n in its L2.
    const uint32_t band = tile / (4 * tiles_m), wide = tiles_n - 4 * band < 4 ? tiles_n - 4 * band : 4, in_band = tile - band * 4 * tiles_m;
    const uint32_t m0 = in_band / wide * BM + (half ? i % 2 * (BM / 2) : 0), n0 = (band * 4 + in_band % wide) * BN;
    if (m0 >= a.M) return;
    if constexpr (HALVES) {
        if (half) return fp8_tile<DT, BM / 2, BN, WM, WN, STAGES>(a, m0, n0, lds);
    }
    fp8_tile<DT, BM, BN, WM, WN, STAGES>(a, m0, n0, lds);
}

uint64_t tiles_of(const Fp8Args& a, uint32_t bm, uint32_t bn) { return (uint64_t)((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn); }

template <int BM, int BN, int WM, int WN, int STAGES, bool HALVES, int... DTS> int launch(int dtype, const Fp8Args& p, uint32_t halved, const LaunchCtx& lc) {
    Fp8Args a = p;
    uint32_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN, whole = (uint32_t)tiles_of(a, BM, BN) - halved;
    const void* fn = nullptr;
    ((dtype == DTS ? (void)(fn = (const void*)fp8_tiles_kernel<DTS, BM, BN, WM, WN, STAGES, HALVES>) : (void)0), ...);
    constexpr size_t lds = STAGES * (BM + BN) * 128 + 2 * BM * kWindow * sizeof(float);
    static_assert(lds <= 160 * 1024, "");
    MTQ_HIP(set_max_dynamic_lds(fn, lds));
    void* args[] = {&a, &tm, &tn, &whole};
    MTQ_HIP(launch_kernel(fn, dim3(whole + 2 * halved), dim3(64 * WM * WN), args, lds, lc));
    return ERR_OK;
}

}  // namespace

// Which tiles a call takes: their number (those cut in two count twice), and threads for each.
enum TileForm { TILES_F32, TILES_64, TILES_128, TILES_256 };
struct TilePick {
    TileForm form;
    uint64_t groups;
    uint32_t threads, halved;
};
static TilePick pick_tiles(int dtype, const Fp8Args& p) {
    if (dtype == DT_F32) return {TILES_F32, tiles_of(p, 128, 128), 256, 0};
    const uint64_t cus = (uint64_t)fp8_num_cus();
    if (tiles_of(p, 128, 64) <= cus) return {TILES_64, tiles_of(p, 128, 64), 512, 0};
    const uint64_t large = tiles_of(p, 256, 256), small = tiles_of(p, 128, 128), over = large % cus;
    // What is over after whole rounds of the CUs is cut in two where that gives each CU one half at most.
    const uint32_t halved = over && 2 * over <= cus ? (uint32_t)over : 0;
    // (the rounds' times as measured, in units of a tenth of a round of small tiles)
    const uint64_t large_time = large / cus * 24 + (halved ? 15 : over ? 24 : 0), small_time = (small + cus - 1) / cus * 10;
    if (large_time < small_time) return {TILES_256, large + halved, 512, halved};
    return {TILES_128, small, 1024, 0};
}

bool fp8_tiles_fit(int dtype, const Fp8Args& p) {
    const TilePick t = pick_tiles(dtype, p);
    return t.groups <= max_workgroups(t.threads);
}

int launch_fp8_tiles(int dtype, const Fp8Args& p, const LaunchCtx& lc) {
    const TilePick t = pick_tiles(dtype, p);
    switch (t.form) {
        case TILES_F32: return launch<128, 128, 2, 2, 2, false, DT_F32>(dtype, p, 0, lc);
        case TILES_64: return launch<128, 64, 4, 2, 4, false, DT_F16, DT_BF16>(dtype, p, 0, lc);
        case TILES_256: return launch<256, 256, 2, 4, 2, true, DT_F16, DT_BF16>(dtype, p, t.halved, lc);
        default: return launch<128, 128, 4, 4, 4, false, DT_F16, DT_BF16>(dtype, p, 0, lc);
    }
}

}  // namespace mtq
