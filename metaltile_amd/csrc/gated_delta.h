// What the kernels of the gated delta rule share. For a sequence's tokens in order and a value head, with S f32 [dv, dk]:
//
//   S = exp(g) S,   u = beta (v - S k),   S += u k^T,   y = scale S q
//
// Heads: value head h reads key head h / (hv / hk). q and k are over their 2-norms first (sqrt(sum of squares + norm_eps)) where norm_eps >= 0.
#pragma once
#include "mtq_device.h"
#include "mtq_internal.h"

namespace mtq {

// The tokens and the state of a sequence. `offsets` are the caller's device memory: whatever they hold, no token outside [0, n_tokens) is
// read or written, and a slot that there is not makes the sequence one that nothing is done for.
struct DeltaSeq {
    uint32_t from, to;    // tokens
    uint32_t slot;
    bool any;
};
__device__ __forceinline__ DeltaSeq delta_seq(const DeltaArgs& a, uint32_t seq) {
    DeltaSeq s;
    if (a.offsets) {
        s.from = min(a.offsets[seq], a.n_tokens);
        s.to = max(s.from, min(a.offsets[seq + 1], a.n_tokens));
    } else {
        const uint32_t each = a.n_tokens / a.n_seqs;
        s.from = seq * each;
        s.to = s.from + each;
    }
    s.slot = a.slots ? a.slots[seq] : seq;
    s.any = s.slot < a.n_slots;
    return s;
}

__device__ __forceinline__ float sum16(float v) { return seg_allreduce(v, 16); }

template <int DT, int DKL, bool WHOLE> __device__ __forceinline__ void load_part(const void* p, size_t i, uint32_t d0, uint32_t dk, float (&v)[DKL]) {
    if constexpr (WHOLE && DKL * (DT == DT_F32 ? 4 : 2) % 16 == 0) {
        constexpr int ES = DT == DT_F32 ? 4 : 2, PER = 16 / ES;
        const uint4* q = (const uint4*)((const char*)p + (i + d0) * ES);
#pragma unroll
        for (int c = 0; c < DKL / PER; c++) {
            const uint4 r = q[c];
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if constexpr (DT == DT_F32) v[c * PER + j] = __uint_as_float(w[j]);
                else {
                    const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
                    v[c * PER + j] = DT == DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < DKL; j++) v[j] = d0 + j < dk ? load_elem<DT>(p, i + d0 + j) : 0.f;
    }
}

// A wave's columns `first` .. first + 3 of head h, over a sequence's tokens one by one.
//
// A wave has four columns of the state (rows of S: dv) in registers, 16 lanes to a column, each with dk / 16 neighbouring values, so that
// the state is read and written in whole lines. Both products with the state use what it was before the token,
//   S k = exp(g) (S0 k),   S q = exp(g) (S0 q) + (k . q) u,
// so that neither waits for the update. A single token is bound by reading and writing the state (64 sequences of 32 heads, dk = dv = 128: 57.7 us
// for 270 MB); many tokens by the seven operations on each of its values, of which the vector units do one a lane and cycle. The next token's
// rows are loaded while one is computed.
//
// DKL: values of k a lane; WHOLE: dk = 16 DKL and every row on 16 bytes.
template <int DT, int DKL, bool WHOLE> __device__ __forceinline__ void delta_tokens(const DeltaArgs& a, const DeltaSeq& s, uint32_t h, uint32_t first) {
    const uint32_t lane = threadIdx.x & 63u;
    if (first >= a.dv) return;
    const uint32_t d0 = (lane & 15u) * DKL, col = first + (lane >> 4);
    const bool in = col < a.dv;
    const uint32_t hk = h / (a.hv / a.hk);
    const size_t state = (((size_t)s.slot * a.hv + h) * a.dv + col) * a.dk;
    // Read before anything else and without a branch, which would wait for it: a column that there is not reads the last one, and a sequence that
    // begins with zeros what state_out holds.
    float S[DKL];
    load_part<DT_F32, DKL, WHOLE>(a.state_in ? a.state_in : a.state_out, in ? state : state - (size_t)(col - a.dv + 1) * a.dk, d0, a.dk, S);
    struct Token {
        float q[DKL], k[DKL], v, g, beta;
    };
    auto load = [&](uint32_t t, Token& x) {
        load_part<DT, DKL, WHOLE>(a.q, (size_t)t * a.q_stride + (size_t)hk * a.dk, d0, a.dk, x.q);
        load_part<DT, DKL, WHOLE>(a.k, (size_t)t * a.k_stride + (size_t)hk * a.dk, d0, a.dk, x.k);
        x.v = load_elem<DT>(a.v, (size_t)t * a.v_stride + (size_t)h * a.dv + (in ? col : a.dv - 1));
        x.g = a.g[(size_t)t * a.hv + h];
        x.beta = a.beta[(size_t)t * a.hv + h];
    };
    Token x;
    if (s.from < s.to) load(s.from, x);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < DKL; j++) S[j] = a.state_in && in ? S[j] : 0.f;
    for (uint32_t t = s.from; t < s.to; t++) {
        Token next = x;
        if (t + 1 < s.to) load(t + 1, next);
        float qq = 0.f, kk = 0.f, qk = 0.f, Sk = 0.f, Sq = 0.f;
#pragma unroll
        for (int j = 0; j < DKL; j++) {
            qq += x.q[j] * x.q[j];
            kk += x.k[j] * x.k[j];
            qk += x.q[j] * x.k[j];
            Sk += S[j] * x.k[j];
            Sq += S[j] * x.q[j];
        }
        qk = sum16(qk);
        float rq = a.scale, rk = 1.f;
        if (a.norm_eps >= 0.f) {
            rq = a.scale / sqrtf(sum16(qq) + a.norm_eps);
            rk = 1.f / sqrtf(sum16(kk) + a.norm_eps);
        }
        const float keep = expf(x.g);
        const float u = x.beta * (x.v - keep * rk * sum16(Sk)), uk = u * rk;
        // (a k whose squares pass f32's range counts as zeros, rk = 0, also where q . k is infinite)
        const float y = rq * (keep * sum16(Sq) + (uk != 0.f ? qk * uk : 0.f));
        if ((lane & 15u) == 0 && in) a.y[((size_t)t * a.hv + h) * a.dv + col] = y;
#pragma unroll
        for (int j = 0; j < DKL; j++) S[j] = keep * S[j] + x.k[j] * uk;
        x = next;
    }
    if (!in) return;
    float* o = a.state_out + state + d0;
    if constexpr (WHOLE && DKL % 4 == 0) {
#pragma unroll
        for (int j = 0; j < DKL; j += 4) *(float4*)(o + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < DKL; j++)
            if (d0 + j < a.dk) o[j] = S[j];
    }
}

// Whether every row of q, k and the states begins on 16 bytes.
inline bool delta_rows_whole(const DeltaArgs& a) {
    const size_t es = a.dtype == DT_F32 ? 4 : 2;
    auto on16 = [&](const void* b, size_t stride) { return (uintptr_t)b % 16 == 0 && stride * es % 16 == 0; };
    return on16(a.q, a.q_stride) && on16(a.k, a.k_stride) && a.dk * es % 16 == 0 && (uintptr_t)a.state_in % 16 == 0 && (uintptr_t)a.state_out % 16 == 0;
}

}  // namespace mtq
