// Softmax attention over a paged cache in packed 4-bit codes (kv_cache.h).
#include "kv_cache.h"

namespace mtq {

namespace {

template <int DT> __device__ __forceinline__ float cached(const KvPart& part, uint64_t at, uint32_t dim, uint32_t group, uint32_t d) {
    const uint32_t word = part.codes[at * (dim / 8) + d / 8];
    const uint64_t g = at * (dim / group) + d / group;
    return fmaf(load_elem<DT>(part.scales, g), (float)(word >> (4 * (d & 7u)) & 15u), load_elem<DT>(part.biases, g));
}

// A wave for each row and query head: a lane scores one token of 64, then has dim / 64 of the values.
template <int DT> __global__ __launch_bounds__(64) void kv_attention_kernel(KvAttentionArgs a) {
    __shared__ float qs[256];
    const KvArgs& kv = a.kv;
    const uint32_t row = blockIdx.x / a.hq, hq = blockIdx.x - row * a.hq, head = hq / (a.hq / kv.hkv), lane = threadIdx.x;
    KvSeq s;
    if (!kv_seq_of(kv, row, s)) return;
    const uint32_t at_row = row - s.first_row, end = at_row + s.len + 1 > s.rows ? s.len + 1 + at_row - s.rows : 0u;   // it sees tokens from .. end - 1
    const uint32_t from = a.window && end > a.window ? end - a.window : 0u;
    for (uint32_t d = lane; d < kv.dim; d += 64) qs[d] = load_elem<DT>(a.q, (uint64_t)row * a.q_stride + (uint64_t)hq * kv.dim + d) * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[4] = {};
    for (uint32_t t0 = from / 64 * 64; t0 < end; t0 += 64) {
        const uint32_t t = t0 + lane;
        const int64_t at = t >= from && t < end ? kv_slot(kv, s.seq, head, t) : -1;
        float x = 0.f;
        if (at >= 0)
            for (uint32_t d = 0; d < kv.dim; d++) x = fmaf(qs[d], cached<DT>(kv.k, (uint64_t)at, kv.dim, kv.group, d), x);
        float top = at >= 0 ? x : -INFINITY;
        for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
        top = fmaxf(top, m);
        if (top == -INFINITY && !__any(at >= 0)) continue;
        const float keep = m == top ? 1.f : __expf(m - top), p = at >= 0 ? __expf(x - top) : 0.f;
        m = top;
        l = l * keep + seg_allreduce(p, 64);
        for (int i = 0; i < 4; i++) o[i] *= keep;
        for (uint32_t j = 0; j < 64; j++) {
            const float pj = __shfl(p, (int)j, 64);
            const int64_t to = (int64_t)((uint64_t)(uint32_t)__shfl((int)((uint64_t)at >> 32), (int)j, 64) << 32 | (uint32_t)__shfl((int)(uint32_t)at, (int)j, 64));
            if (to < 0) continue;
            for (uint32_t i = 0; i < kv.dim / 64; i++) o[i] = fmaf(pj, cached<DT>(kv.v, (uint64_t)to, kv.dim, kv.group, lane + 64 * i), o[i]);
        }
    }
    for (uint32_t i = 0; i < kv.dim / 64; i++) store_elem<DT>(a.out, (uint64_t)row * a.out_stride + (uint64_t)hq * kv.dim + lane + 64 * i, l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

int launch_kv_attention(int dtype, const KvAttentionArgs& p, const LaunchCtx& lc) {
    KvAttentionArgs a = p;
    const uint64_t groups = (uint64_t)a.kv.n_tokens * a.hq;
    if (groups > max_workgroups(64)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    const void* fn[] = {(const void*)kv_attention_kernel<DT_F32>, (const void*)kv_attention_kernel<DT_F16>, (const void*)kv_attention_kernel<DT_BF16>};
    void* args[] = {&a};
    MTQ_HIP(launch_kernel(fn[dtype], dim3((uint32_t)groups), dim3(64), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
