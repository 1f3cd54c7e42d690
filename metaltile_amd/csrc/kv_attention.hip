// Which kernel a call of the attention over the 4-bit cache takes, how its tokens are cut, and the slices' sums joined.
#include "kv_attention.h"

namespace mtq {

namespace {

// A wave for each row and query head: its slices joined.
// Rows outside all sequences are left alone.
__device__ __forceinline__ bool kv_of_some_sequence(const KvArgs& kv, uint32_t row) {
    return row < kv.n_tokens && (!kv.offsets || (row >= kv.offsets[0] && row < kv.offsets[kv.n_seqs]));
}

// Up to eight slices: sixteen lanes to a row of a head, so four of them to a wave (60000 rows of 64 values in up to three slices: 21 us with a wave each, most of it
// latency). All loads of a row's values go out together.
constexpr uint32_t kJoinMost = 8;
template <int DT, int D> __global__ __launch_bounds__(256) void kv_join_kernel(KvAttentionArgs a, KvParts parts) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, at = blockIdx.x * 16u + threadIdx.x / 16u, row = at / a.hq, h = at - row * a.hq;
    const bool in = row < a.kv.n_tokens;
    const float* sums = parts.sums + (uint64_t)(in ? at : 0u) * parts.slices * 2;
    const float bar = l < parts.slices ? sums[2 * l] : -INFINITY, part = l < parts.slices ? sums[2 * l + 1] : 0.f;
    const uint32_t end = (uint32_t)(__ballot(part == kNoMore) >> (lane & 48u)) & 0xFFFFu, n = end ? (uint32_t)__builtin_ctz(end) : parts.slices;
    float top = l < n ? bar : -INFINITY;
#pragma unroll
    for (int i = 1; i < 16; i <<= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
    const float f = l >= n ? 0.f : bar == -INFINITY ? (part == 0.f ? 0.f : 1.f) : exp2f(bar - top);
    const bool none = l >= n || (f == 0.f && part == 0.f);   // (its values are nothing, or not there)
    float total = none ? 0.f : part * f;
#pragma unroll
    for (int i = 1; i < 16; i <<= 1) total += __shfl_xor(total, i, 64);
    const uint32_t there = (uint32_t)(__ballot(!none) >> (lane & 48u)) & 0xFFFFu;
    if (n == 0 || !kv_of_some_sequence(a.kv, row)) return;   // (of one slice: written already)
    const float* values = parts.values + (uint64_t)at * parts.slices * D + 4 * l;
    kr_f32x4 v[D / 64] = {};
#pragma unroll
    for (uint32_t i0 = 0; i0 < kJoinMost; i0 += 4) {
        if (i0 >= n) break;
        kr_f32x4 x[4][D / 64];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < D / 64; j++) x[i][j] = *(const kr_f32x4*)(values + (uint64_t)(i0 + i < n ? i0 + i : n - 1u) * D + 64 * j);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const float by = __shfl(f, (int)((lane & 48u) + i0 + i), 64);
            if (there >> (i0 + i) & 1u) {
#pragma unroll
                for (int j = 0; j < D / 64; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) v[j][e] = fmaf(x[i][j][e], by, v[j][e]);
            }
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int j = 0; j < D / 64; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) store_elem<DT>(a.out, (uint64_t)row * a.out_stride + (uint64_t)h * D + 64 * j + 4 * l + e, total == 0.f ? 0.f : v[j][e] * inv);
}

// More of them: a workgroup to a row of a head, D / 4 lanes to a slice's numbers. The slices' loads go out together: with a branch on a slice's sum between them,
// 32 slices took 15 us.
template <int DT, int D> __global__ __launch_bounds__(256) void kv_join_many_kernel(KvAttentionArgs a, KvParts parts) {
    constexpr uint32_t LANES = D / 4, TURNS = 256 / LANES;
    __shared__ kr_f32x4 others[TURNS][LANES + 1];   // (values; sum)
    const uint32_t lane = threadIdx.x & 63u, at = blockIdx.x, row = at / a.hq, h = at - row * a.hq, turn = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
    const float* sums = parts.sums + (uint64_t)at * parts.slices * 2;
    const float* values = parts.values + (uint64_t)at * parts.slices * D + d;
    uint32_t n = parts.slices;
    float top = -INFINITY;
    for (uint32_t i = lane; i - lane < n; i += 64) {
        const float bar = i < n ? sums[2 * i] : -INFINITY, part = i < n ? sums[2 * i + 1] : 0.f;
        const uint64_t no_more = __ballot(part == kNoMore);
        if (no_more) n = i - lane + (uint32_t)__builtin_ctzll(no_more);
        if (i < n) top = fmaxf(top, bar);
    }
    if (n == 0 || !kv_of_some_sequence(a.kv, row)) return;   // (of one slice: written already)
    for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
    float total = 0.f;
    kr_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t i = turn; i < n; i += TURNS) {
        const float bar = sums[2 * i], part = sums[2 * i + 1], f = bar == -INFINITY ? (part == 0.f ? 0.f : 1.f) : exp2f(bar - top);
        const kr_f32x4 x = *(const kr_f32x4*)(values + (uint64_t)i * D);
        const bool none = f == 0.f && part == 0.f;   // (its values are nothing, or not there)
        total = fmaf(part, f, total);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = none ? v[j] : fmaf(x[j], f, v[j]);
    }
    others[turn][d / 4] = v;
    if (d == 0) others[turn][LANES][0] = total;
    __syncthreads();
    if (turn) return;
#pragma unroll
    for (uint32_t i = 1; i < TURNS; i++) {
        total += others[i][LANES][0];
        v += others[i][d / 4];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) store_elem<DT>(a.out, (uint64_t)row * a.out_stride + (uint64_t)h * D + d + j, total == 0.f ? 0.f : v[j] / total);
}

}  // namespace

int launch_kv_join(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    KvAttentionArgs a = p;
    KvParts q = parts;
#define MTQ_KV_JOIN(DT, D) {(const void*)kv_join_kernel<DT, D>, (const void*)kv_join_many_kernel<DT, D>}
#define MTQ_KV_JOINS(DT) {MTQ_KV_JOIN(DT, 64), MTQ_KV_JOIN(DT, 128), MTQ_KV_JOIN(DT, 256)}
    const void* fn[3][3][2] = {MTQ_KV_JOINS(DT_F32), MTQ_KV_JOINS(DT_F16), MTQ_KV_JOINS(DT_BF16)};
#undef MTQ_KV_JOIN
#undef MTQ_KV_JOINS
    const bool many = parts.slices > kJoinMost;
    const uint64_t rows = (uint64_t)a.kv.n_tokens * a.hq, groups = many ? rows : (rows + 15) / 16;
    if (groups > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    void* args[] = {&a, &q};
    MTQ_HIP(launch_kernel(fn[dtype][a.kv.dim == 64 ? 0 : a.kv.dim == 128 ? 1 : 2][many], dim3((uint32_t)groups), dim3(256), args, 0, lc));
    return ERR_OK;
}

static uint32_t num_cus() {
    static int n = 0;
    if (n == 0) {
        int dev = 0, v = 0;
        n = (hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) ? v : 256;
    }
    return (uint32_t)n;
}

// Rows are new tokens times the query heads that share a key head, for each sequence on average:
//   to 4     the kernel with a token to a lane, where heads have 128 values or more and there is work for the card (64 sequences of 4096 tokens, 4 rows, bf16: 70 us
//            against 74 of the one below, f16 70 / 85, in groups of 32 80 / 108, 256 values 123 / 132; 64 values 67 / 50, one sequence of 1000 tokens 13.4 / 12.1)
//   to 128   the one with 16 rows to a wave, where sequences and heads fill the card (32 sequences of 4096 tokens, 128 rows: 264 us against 360 of the one below, 64 rows
//            147 / 366), else to 64 (4 of 2048 tokens, 128 rows 62 / 41, 64 rows 35 / 34); f32 to half of
//            that (64 rows 244 / 417, 128 rows 466 / 412; 32 rows 27 / 32, 64 rows 45 / 33)
//   above    f16 and bf16: keys and values laid out in T first (256 rows: 494 / 372 and 115 / 45; a prompt of 8192 tokens 531 us against 942 of the next). It has to have
//            scratch for as many tokens as max_len allows, up to 1 GiB; f32, and calls without: the codes as they are
KvPlan kv_attention_plan(int dtype, const KvAttentionArgs& a) {
    KvPlan p;
    const uint64_t cus = num_cus(), rows = (uint64_t)a.kv.n_tokens * (a.hq / a.kv.hkv), n_seqs = a.kv.n_seqs;
    const uint64_t row_bytes = (uint64_t)a.kv.n_tokens * a.hq * (a.kv.dim + 2) * sizeof(float), most_bytes = (uint64_t)64 << 20;   // of a slice; of all
    const uint32_t span = a.window && a.window < a.kv.max_len ? a.window : a.kv.max_len;   // tokens that a row sees at most
    const uint64_t images = ((uint64_t)a.kv.max_len + kBlock - 1) / kBlock * n_seqs * a.kv.hkv * (128ull * a.kv.dim + 4);
    const bool prompts = dtype != DT_F32 && images && images <= (1ull << 30);
    const bool filled = n_seqs * a.kv.hkv * span >= 2048 * cus, few = a.kv.dim >= 128 && filled;
    p.kernel = options().kv_kernel ? options().kv_kernel : few && rows <= 4 * n_seqs ? 3 : rows <= (filled ? 128 : 64) / (dtype == DT_F32 ? 2 : 1) * n_seqs ? 1 : prompts ? 4 : 2;
    if (p.kernel == 4 && !prompts) p.kernel = 2;
    if (p.kernel == 3 && a.kv.dim < 128) p.kernel = 1;
    if (p.kernel == 4) p.images = (size_t)((images + 255) / 256 * 256);
    uint64_t slices, pieces;
    if (p.kernel == 2 || p.kernel == 4) {
        // Two tiles' worth of workgroups to a compute unit; the grid has room for twice that, since tiles that see little are not cut. Less than 256 tokens to a
        // slice do not pay for what goes through memory (a prompt of 512 tokens in slices of 256: 26 us, whole 23).
        const uint64_t groups = (rows / (p.kernel == 4 ? kv_prompt_rows(a.kv.dim) : kv_tile_rows(dtype, a.kv.dim)) + n_seqs) * a.kv.hkv, want = (4 * cus + groups - 1) / groups;
        slices = span < 1024 ? 1 : want < span / 256 ? want : span / 256;
        pieces = 2 * cus / a.kv.hkv;
        p.least = 8;
        if (options().kv_slices) {
            slices = (uint64_t)options().kv_slices;
            pieces = 0xFFFFFFFFu;
            p.least = 1;
        }
        while (slices > 1 && groups * slices > max_workgroups(512)) slices--;
    } else {
        // The same, and no piece longer than two of a sequence's average. Where sequences and heads fill the card as they come they are not cut: from three to a compute unit on
        // while no sequence is long, else from eight, since one that is ends alone. 128 sequences of 1 to 1000 tokens, 16 rows: 34.8 us, cut 36.4, f32 heads of 64 values 26.9 / 29.1;
        // of 1 to 4096 103.7 / 93.5 and 81.6 / 76.4, of 1 to 8192 with four rows of f32 266 / 210. Four rows in 16 bits, to 4096: 84 / 87 and with 64 values 52.5 / 49.1, even
        // ones 126 / 132 and 75.5 / 81; to 8192 149 / 132.
        const uint64_t seen = (uint64_t)span + a.kv.n_tokens < a.kv.max_len ? (uint64_t)span + a.kv.n_tokens : a.kv.max_len, blocks = (seen + 63) / 64;   // by all rows of a sequence
        pieces = 2 * cus / a.kv.hkv > n_seqs / 2 ? 2 * cus / a.kv.hkv : n_seqs / 2;
        const uint64_t most = blocks < 10 ? 1 : blocks / (p.kernel == 3 ? 4 : 2);   // (a step of 64 or 32 tokens for each wave: 2000 tokens 10.7 us, of twice that 11.9; 640 tokens uncut 10.9)
        slices = most < pieces ? most : pieces;
        if (n_seqs * a.kv.hkv >= (blocks <= (dtype != DT_F32 && rows <= 4 * n_seqs ? 64u : 32u) ? 3 : 8) * cus) slices = 1;
        if (options().kv_slices) {
            slices = (uint64_t)options().kv_slices;
            pieces = slices * n_seqs;
        }
        const uint64_t sets = kv_sets<4>(a);   // (or fewer)
        if (n_seqs > kCutSeqs || sets * blocks >= 1ull << 32) slices = 1;
        while (slices > 1 && (sets + pieces) * a.kv.hkv > max_workgroups(256)) {
            pieces /= 2;
            slices = slices < pieces ? slices : pieces;
        }
        if (slices > most_bytes / row_bytes) slices = most_bytes / row_bytes;
        if (slices < 1) slices = 1;
        p.least = (uint32_t)((blocks + slices - 1) / slices);   // (of what max_len allows, so a short sequence under a large max_len has few pieces: 1000 tokens under 131072 take 16.6 us, under 1000 10.7)
    }
    if (slices > most_bytes / row_bytes) slices = most_bytes / row_bytes;
    p.slices = slices < 1 ? 1 : (uint32_t)slices;
    p.pieces = pieces ? (uint32_t)pieces : 1;
    p.scratch = p.images + (p.slices > 1 ? (size_t)(row_bytes * p.slices) : 0);
    return p;
}

int launch_kv_attention(int dtype, const KvAttentionArgs& a, const KvPlan& plan, void* scratch, const LaunchCtx& lc) {
    if ((uint64_t)a.kv.n_seqs * a.kv.hkv > max_workgroups(256)) return fail(ERR_SHAPE, "more sequences and heads than a launch can have workgroups");
    KvParts parts;
    KvImages images;
    if (scratch) {
        images.blocks = (a.kv.max_len + kBlock - 1) / kBlock;
        images.data = (uint8_t*)scratch;
        images.flags = (uint32_t*)(images.data + (size_t)images.blocks * a.kv.n_seqs * a.kv.hkv * (128 * a.kv.dim));
        parts.slices = plan.slices;
        parts.pieces = plan.pieces;
        parts.least = plan.least;
        parts.values = (float*)((char*)scratch + plan.images);
        parts.sums = parts.values + (size_t)a.kv.n_tokens * a.hq * parts.slices * a.kv.dim;
    }
    switch (plan.kernel) {
        case 1: return launch_kv_rows(dtype, a, parts, lc);
        case 3: return launch_kv_quads(dtype, a, parts, lc);
        case 4:
            if (scratch) return launch_kv_prompts(dtype, a, parts, images, lc);
    }
    return launch_kv_tiles(dtype, a, parts, lc);
}

}  // namespace mtq
