// Which kernel a call of the attention over the 4-bit cache takes, and into how many slices its tokens are cut.
#include "kv_attention.h"

namespace mtq {

namespace {

// A wave for each row and query head: its slices joined.
template <int DT, int D> __global__ __launch_bounds__(256) void kv_join_kernel(KvAttentionArgs a, KvParts parts) {
    const uint32_t lane = threadIdx.x & 63u, at = blockIdx.x * 4 + (threadIdx.x >> 6), row = at / a.hq, h = at - row * a.hq;
    if (row >= a.kv.n_tokens) return;
    KvSeq s;
    if (!kv_seq_of(a.kv, row, s)) return;
    const float* sums = parts.sums + (uint64_t)at * parts.slices * 2;
    float top = -INFINITY;
    for (uint32_t i = lane; i < parts.slices; i += 64) top = fmaxf(top, sums[2 * i]);
    for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
    float total = 0.f, v[D / 64] = {};
    for (uint32_t i = 0; i < parts.slices; i++) {
        const float bar = sums[2 * i], part = sums[2 * i + 1], f = bar == -INFINITY ? (part == 0.f ? 0.f : 1.f) : exp2f(bar - top);
        if (f == 0.f && part == 0.f) continue;
        total = fmaf(part, f, total);
#pragma unroll
        for (int j = 0; j < D / 64; j++) v[j] = fmaf(parts.values[((uint64_t)at * parts.slices + i) * D + lane + 64 * j], f, v[j]);
    }
#pragma unroll
    for (int j = 0; j < D / 64; j++) store_elem<DT>(a.out, (uint64_t)row * a.out_stride + (uint64_t)h * D + lane + 64 * j, total == 0.f ? 0.f : v[j] / total);
}

}  // namespace

int launch_kv_join(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    KvAttentionArgs a = p;
    KvParts q = parts;
    const void* fn[3][3] = {{(const void*)kv_join_kernel<DT_F32, 64>, (const void*)kv_join_kernel<DT_F32, 128>, (const void*)kv_join_kernel<DT_F32, 256>},
                            {(const void*)kv_join_kernel<DT_F16, 64>, (const void*)kv_join_kernel<DT_F16, 128>, (const void*)kv_join_kernel<DT_F16, 256>},
                            {(const void*)kv_join_kernel<DT_BF16, 64>, (const void*)kv_join_kernel<DT_BF16, 128>, (const void*)kv_join_kernel<DT_BF16, 256>}};
    const uint64_t groups = ((uint64_t)a.kv.n_tokens * a.hq + 3) / 4;
    if (groups > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    void* args[] = {&a, &q};
    MTQ_HIP(launch_kernel(fn[dtype][a.kv.dim == 64 ? 0 : a.kv.dim == 128 ? 1 : 2], dim3((uint32_t)groups), dim3(256), args, 0, lc));
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

KvPlan kv_attention_plan(int dtype, const KvAttentionArgs& a) {
    KvPlan p;
    const uint64_t units = (uint64_t)a.kv.n_seqs * a.kv.hkv, cus = num_cus(), rows = (uint64_t)a.kv.n_tokens * (a.hq / a.kv.hkv);
    const uint32_t span = a.window && a.window < a.kv.max_len ? a.window : a.kv.max_len;   // tokens that a row sees at most
    p.tiles = rows > 32ull * a.kv.n_seqs;
    if (options().kv_kernel) p.tiles = options().kv_kernel == 2;
    uint64_t groups;   // of one slice
    if (p.tiles) {
        groups = (rows / kv_tile_rows(dtype, a.kv.dim) + a.kv.n_seqs) * a.kv.hkv;
        const uint64_t want = (cus + groups - 1) / groups, most = span / 512;
        p.slices = (uint32_t)(want < most ? want : most);
    } else {
        groups = units;
        p.large = units < 2 * cus;
        const uint64_t want = ((p.large ? 1 : 4) * cus + units - 1) / units, most = span / (p.large ? 1024 : 512);
        p.slices = (uint32_t)(want < most ? want : most);
    }
    if (options().kv_waves) p.large = options().kv_waves == 2;
    if (options().kv_slices) p.slices = (uint32_t)options().kv_slices;
    if (p.slices < 1) p.slices = 1;
    while (p.slices > 1 && groups * p.slices > max_workgroups(1024)) p.slices--;
    p.scratch = p.slices > 1 ? (size_t)a.kv.n_tokens * a.hq * p.slices * (a.kv.dim + 2) * sizeof(float) : 0;
    return p;
}

int launch_kv_attention(int dtype, const KvAttentionArgs& a, const KvPlan& plan, void* scratch, const LaunchCtx& lc) {
    KvParts parts;
    parts.slices = scratch ? plan.slices : 1;
    parts.values = (float*)scratch;
    parts.sums = scratch ? parts.values + (size_t)a.kv.n_tokens * a.hq * parts.slices * a.kv.dim : nullptr;
    if ((uint64_t)a.kv.n_seqs * a.kv.hkv * parts.slices > max_workgroups(1024)) return fail(ERR_SHAPE, "more sequences and heads than a launch can have workgroups");
    return plan.tiles ? launch_kv_tiles(dtype, a, parts, lc) : launch_kv_rows(dtype, a, parts, plan.large, lc);
}

}  // namespace mtq
