// Writer and reader of a paged cache in packed 4-bit codes (kv_cache.h): memory bounds both, eight values a lane, 16 bytes of 16-bit elements
// on one side and a word of codes on the other.
#include "kv_cache.h"

// Every a*b+c here is two rounded operations, as the packed format's quantiser has them: a code is the same wherever it is made.
#pragma STDC FP_CONTRACT OFF

namespace mtq {

namespace {

template <int DT> __device__ __forceinline__ void kv_load8(const void* p, uint64_t i, float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 r = *(const uint4*)((const uint16_t*)p + i);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
            v[j] = DT == DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}
template <int DT> __device__ __forceinline__ void kv_store8(void* p, uint64_t i, const float (&v)[8]) {
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

// Values e0 .. e0 + 7 of a head at p + i, turned by the table's row.
template <int DT> __device__ __forceinline__ void kv_turned8(const KvAppendArgs& a, const void* p, uint64_t i, uint32_t e0, uint32_t place, float (&v)[8]) {
#pragma clang fp contract(off)
    kv_load8<DT>(p, i + e0, v);
    if (e0 >= a.rot) return;
    const float* row = a.cos_sin + (uint64_t)place * a.rot;
    const uint32_t half = a.rot / 2;
    if (a.neighbours) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if (e0 + j >= a.rot) break;
            const float c = row[(e0 + j) / 2], s = row[half + (e0 + j) / 2], x = v[j], y = v[j + 1];
            const float xc = x * c, ys = y * s, yc = y * c, xs = x * s;
            v[j] = xc - ys;
            v[j + 1] = yc + xs;
        }
    } else if (a.rot % 16 == 0) {   // (all eight are in one half)
        const bool upper = e0 >= half;
        const uint32_t j0 = upper ? e0 - half : e0;
        float o[8], c[8], s[8];
        kv_load8<DT>(p, i + (upper ? j0 : e0 + half), o);
        kv_load8<DT_F32>(row, j0, c);
        kv_load8<DT_F32>(row, half + j0, s);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float mine = v[j] * c[j], other = o[j] * s[j];
            v[j] = upper ? mine + other : mine - other;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t e = e0 + j;
            if (e >= a.rot) continue;
            const bool upper = e >= half;
            const uint32_t at = upper ? e - half : e;
            const float o = load_elem<DT>(p, i + (upper ? at : e + half));
            const float mine = v[j] * row[at], other = o * row[half + at];
            v[j] = upper ? mine + other : mine - other;
        }
    }
}

// A lane has eight values of a head of one of the call's rows: the query heads, then key heads, then value heads. All loads of a wave come before its
// stores, and a head is within a wave: queries may be turned in place.
template <int DT> __global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, uint32_t groups_per_row) {
#pragma clang fp contract(off)
    const KvArgs& kv = a.kv;
    const uint32_t row = blockIdx.x / groups_per_row, unit = (blockIdx.x - row * groups_per_row) * 256 + threadIdx.x;
    KvSeq s;
    if (!kv_seq_of(kv, row, s)) return;
    const uint32_t words = kv.dim / 8, at_row = row - s.first_row;
    if (at_row + s.len < s.rows) return;   // no place
    const uint32_t place = s.len - s.rows + at_row, slot = unit / words, e0 = (unit - slot * words) * 8;   // (dim is a power of two times 8)
    if (slot >= a.hq + 2 * kv.hkv) return;   // (whole heads)
    float v[8];
    if (slot < a.hq) {
        kv_turned8<DT>(a, a.q, (uint64_t)row * a.q_stride + (uint64_t)slot * kv.dim, e0, place, v);
        kv_store8<DT>(a.q_out, (uint64_t)row * a.q_out_stride + (uint64_t)slot * kv.dim + e0, v);
        return;
    }
    const bool value = slot >= a.hq + kv.hkv;
    const uint32_t head = slot - a.hq - (value ? kv.hkv : 0u);
    if (value) kv_load8<DT>(a.v, (uint64_t)row * a.v_stride + (uint64_t)head * kv.dim + e0, v);
    else kv_turned8<DT>(a, a.k, (uint64_t)row * a.k_stride + (uint64_t)head * kv.dim, e0, place, v);
    float mn = v[0], mx = v[0];
    bool fine = true;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        fine = fine && fabsf(v[j]) < INFINITY;
        mn = v[j] < mn ? v[j] : mn;
        mx = v[j] > mx ? v[j] : mx;
    }
    uint32_t all_fine = fine;
    for (uint32_t d = 1; d < kv.group / 8; d <<= 1) {   // (a group's lanes are neighbours and within a head)
        const float omn = __shfl_xor(mn, (int)d, 64), omx = __shfl_xor(mx, (int)d, 64);
        mn = omn < mn ? omn : mn;
        mx = omx > mx ? omx : mx;
        all_fine &= (uint32_t)__shfl_xor((int)all_fine, (int)d, 64);
    }
    float scale = (mx - mn) / 15.0f;
    if (scale < 1.0e-7f) scale = 1.0f;
    const float inv = 1.0f / scale;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float d = v[j] - mn;
        const float p = d * inv;
        float q = p + 0.5f;
        q = q < 0.0f ? 0.0f : q;
        q = q > 15.0f ? 15.0f : q;
        word |= (uint32_t)q << (4 * j);
    }
    if (!all_fine) {   // reads as NaN, all of it
        scale = mn = __builtin_nanf("");
        word = 0;
    }
    const int64_t to = kv_slot(kv, s.seq, head, place);
    if (to < 0) return;
    (value ? kv.v.codes : kv.k.codes)[(uint64_t)to * words + e0 / 8] = word;
    if (e0 % kv.group == 0) {
        const uint64_t g = (uint64_t)to * (kv.dim / kv.group) + e0 / kv.group;
        store_elem<DT>(value ? kv.v.scales : kv.k.scales, g, scale);
        store_elem<DT>(value ? kv.v.biases : kv.k.biases, g, mn);
    }
}

// A lane has a word of codes: of keys, or in the launch's second half of values.
template <int DT> __global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a, uint32_t groups_per_row) {
#pragma clang fp contract(off)
    const KvArgs& kv = a.kv;
    const uint32_t row = blockIdx.x / groups_per_row, unit = (blockIdx.x - row * groups_per_row) * 256 + threadIdx.x;
    KvSeq s;
    if (!kv_seq_of(kv, row, s)) return;
    const uint32_t words = kv.dim / 8, at_row = row - s.first_row;
    if (at_row + s.len < s.rows) return;
    const uint32_t place = s.len - s.rows + at_row, head = unit / words, e0 = (unit - head * words) * 8;
    if (head >= kv.hkv) return;
    const int64_t from = kv_slot(kv, s.seq, head, place);
    if (from < 0) return;
    const uint32_t* codes = blockIdx.y ? kv.v.codes : kv.k.codes;
    const void *scales = blockIdx.y ? kv.v.scales : kv.k.scales, *biases = blockIdx.y ? kv.v.biases : kv.k.biases;
    void* out = blockIdx.y ? a.v : a.k;
    if (!out) return;
    const uint64_t g = (uint64_t)from * (kv.dim / kv.group) + e0 / kv.group;
    const uint32_t word = codes[(uint64_t)from * words + e0 / 8];
    const float scale = load_elem<DT>(scales, g), bias = load_elem<DT>(biases, g);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float p = scale * (float)(word >> (4 * j) & 15u);
        v[j] = p + bias;
    }
    kv_store8<DT>(out, ((uint64_t)row * kv.hkv + head) * kv.dim + e0, v);
}

}  // namespace

int launch_kv_append(int dtype, const KvAppendArgs& p, const LaunchCtx& lc) {
    KvAppendArgs a = p;
    uint32_t per_row = (uint32_t)(((uint64_t)(a.hq + 2 * a.kv.hkv) * (a.kv.dim / 8) + 255) / 256);
    const uint64_t groups = (uint64_t)per_row * a.kv.n_tokens;
    if (groups > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    const void* fn[] = {(const void*)kv_append_kernel<DT_F32>, (const void*)kv_append_kernel<DT_F16>, (const void*)kv_append_kernel<DT_BF16>};
    void* args[] = {&a, &per_row};
    MTQ_HIP(launch_kernel(fn[dtype], dim3((uint32_t)groups), dim3(256), args, 0, lc));
    return ERR_OK;
}

int launch_kv_read(int dtype, const KvReadArgs& p, const LaunchCtx& lc) {
    KvReadArgs a = p;
    uint32_t per_row = (uint32_t)(((uint64_t)a.kv.hkv * (a.kv.dim / 8) + 255) / 256);
    const uint64_t groups = (uint64_t)per_row * a.kv.n_tokens;
    if (groups > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    const void* fn[] = {(const void*)kv_read_kernel<DT_F32>, (const void*)kv_read_kernel<DT_F16>, (const void*)kv_read_kernel<DT_BF16>};
    void* args[] = {&a, &per_row};
    MTQ_HIP(launch_kernel(fn[dtype], dim3((uint32_t)groups, 2), dim3(256), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
