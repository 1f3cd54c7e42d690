// The gated delta rule (gated_delta.h) in chunks of 64 tokens, on the matrix cores.
//
// With G_t the sum of g over a chunk's tokens up to t, r_t and q_t's factor p_t = scale r'_t the norms' reciprocals (1 without them), and S0
// the state before the chunk, the recurrence of the chunk's 64 updates u_t is one triangular system:
//
//   (1 + A) U = diag(beta) (V - diag(e^G r) K S0),    A_ts = beta_t r_t r_s e^(G_t - G_s) (k_t . k_s), s < t
//   Y = diag(e^G p) Q S0 + P U,                       P_ts = p_t r_s e^(G_t - G_s) (q_t . k_s), s <= t
//   S1 = e^(G_63) S0 + K^T diag(r e^(G_63 - G)) U
//
// Two launches. The first, a workgroup to a chunk and key head, works out what does not depend on the state: P and T = (1 + A)^-1 diag(beta)
// (16 x 16 blocks on the diagonal by substitution, the rest from pairs of blocks: [A 0; C B]^-1 = [A' 0; -B' C A' B']). The second walks a
// sequence's chunks in order, a workgroup to a head and 16 columns of the state: U = T (V - ..), Y and S1. Half of its waves carry what the
// next chunk waits for (K S0, U), the others Q S0 and P U beside them; all update the state.
//
// Everything is held in f32 and multiplied as bf16 on the matrix cores without losing it: an f32 value is the sum of three bf16 terms (8
// bits each, by rounding and taking the rest), a bf16 q or k is one, an f16 one two. Of the products of terms those of 2^-24 and less of the
// whole are left out: 3 products for bf16 q and k against f32, 5 for f16, 6 for f32 against f32. That is f32 arithmetic at the rate of the
// matrix cores over 3 to 6, two to five times what their own f32 instructions do. (Terms end at 2^-133, bf16's smallest: of values under about
// 2^-109 the last bits are lost.) Sums of decays are f64 (differences of far ones would lose an f32's last digits).
//
// What the first launch leaves for the second lies in the order in which lanes hand it to the matrix cores, 16 bytes a lane, so that the
// walk reads whole lines into registers and waits for no transposition.
#include "gated_delta.h"
#include "mfma16.h"

namespace mtq {

namespace {

constexpr uint32_t kChunk = 64;
constexpr uint32_t kFewTokens = 16;       // sequences up to this length go token by token
constexpr uint32_t kTriBytes = 6 * 3 * 1024;   // T or P: 6 steps of 16 x 32 that hold any of the triangle, three terms
constexpr uint32_t kHeadBytes = 2 * kTriBytes + 1024;   // a value head's T, P, and four rows of 64 f32: e^G r, e^G p, r e^(G_63 - G), e^(G_63)

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct ChunkArgs {
    DeltaArgs d;
    uint8_t* scratch;
    uint32_t lo, hi;        // this launch's slots for chunks: sequence i's chunk c has slot first_slot(i) + c
    uint32_t by_tokens;     // how slots are numbered
    uint32_t whole;         // rows of q and k on 16 bytes
    uint32_t parts;         // workgroups of the first launch for a chunk and key head
};

template <int DKP, int NT> struct Layout {
    static constexpr uint32_t kOp = NT * kChunk * DKP * 2;      // K, Q or K^T of a key head
    static constexpr uint32_t kKeyBytes = 3 * kOp;
    static __device__ __host__ size_t slot_bytes(uint32_t hk, uint32_t hv) { return (size_t)hk * kKeyBytes + (size_t)hv * kHeadBytes; }
};

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    typedef __attribute__((ext_vector_type(8))) __bf16 v8;
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
// The sum of products of terms i and j with i + j < MOST: small ones first.
template <int NA, int NB> __device__ __forceinline__ f32x4 mfma_terms(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c) {
    constexpr int MOST = 3;
#pragma unroll
    for (int s = MOST - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++)
            if (s - i >= 0 && s - i < NB) c = mfma_bf16(a[i], b[s - i], c);
    return c;
}

// The same onto several sums in turn, so that an instruction does not wait for the one before: sum number `at`, at + 1, .. of N.
template <int NA, int NB, int N> __device__ __forceinline__ void mfma_terms_on(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 (&c)[N], int at) {
    constexpr int MOST = 3;
#pragma unroll
    for (int s = MOST - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++)
            if (s - i >= 0 && s - i < NB) {
                c[at % N] = mfma_bf16(a[i], b[s - i], c[at % N]);
                at++;
            }
}

// v as N bf16 terms, two values to a word: term k of (v0, v1) in w[k].
template <int N> __device__ __forceinline__ void terms(float v0, float v1, uint32_t (&w)[N]) {
    typedef __attribute__((ext_vector_type(2))) float f32x2;
#pragma unroll
    for (int k = 0; k < N; k++) {
        w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v0, v1}), bf16x2_t));
        v0 -= __uint_as_float(w[k] << 16);
        v1 -= __uint_as_float(w[k] & 0xFFFF0000u);
    }
}
template <int N> __device__ __forceinline__ void terms8(const float (&v)[8], u32x4 (&w)[N]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t t[N];
        terms<N>(v[2 * j], v[2 * j + 1], t);
#pragma unroll
        for (int k = 0; k < N; k++) w[k][j] = t[k];
    }
}

template <int DT> __device__ __forceinline__ void load8(const void* p, size_t i, uint32_t d, uint32_t dk, bool whole, float (&v)[8]) {
    if (whole && d + 8 <= dk) {
        load_part<DT, 8, true>(p, i, d, dk, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = d + j < dk ? load_elem<DT>(p, i + d + j) : 0.f;
    }
}

// A sequence's first slot, in one of two numberings of which a call takes the one with fewer slots: from / 64 + seq, which gives every sequence a
// slot, or by tokens alone, from / 17: a sequence that takes chunks has 17 tokens or more, and floor(n / 17) >= ceil(n / 64) for those, so the next one
// begins behind its last slot (256 sequences of two tokens: 31 slots instead of 264, which are 2 MB each with 16 and 32 heads of 128 bf16).
constexpr uint32_t kFewestChunked = kFewTokens + 1;
__device__ __host__ __forceinline__ uint32_t first_slot(uint32_t from, uint32_t seq, uint32_t by_tokens) {
    return by_tokens ? from / kFewestChunked : from / kChunk + seq;
}
// Slots of a call; `by_tokens`: in which numbering.
inline uint64_t slots_of(const DeltaArgs& d, uint32_t& by_tokens) {
    const uint64_t with = (uint64_t)d.n_tokens / kChunk + d.n_seqs, tokens = (uint64_t)d.n_tokens / kFewestChunked + 1;
    by_tokens = tokens < with;
    return by_tokens ? tokens : with;
}
// The sequence that a slot belongs to: the last whose first slot is not behind it.
__device__ __forceinline__ uint32_t seq_of(const ChunkArgs& c, uint32_t slot) {
    const DeltaArgs& a = c.d;
    if (!a.offsets) {   // (equal lengths: no memory to be read)
        uint32_t lo = 0, hi = a.n_seqs;
        const uint32_t each = a.n_tokens / a.n_seqs;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (first_slot(mid * each, mid, c.by_tokens) <= slot) lo = mid;
            else hi = mid;
        }
        return lo;
    }
    // 64 sequences at a time, so that a few reads of memory after one another find it: those whose first slot is not behind it come first
    uint32_t lo = 0, step = 1;
    while (step * 64 < a.n_seqs) step *= 64;   // (sequences are less than 2^24)
    for (;; step /= 64) {
        const uint32_t i = lo + (threadIdx.x & 63u) * step;
        const bool before = i < a.n_seqs && first_slot(min(a.offsets[i < a.n_seqs ? i : 0], a.n_tokens), i, c.by_tokens) <= slot;
        const uint32_t n = (uint32_t)__popcll(__ballot(before));
        if (n) lo += (n - 1) * step;
        if (step == 1) return lo;
    }
}

constexpr int kPitch = 68;   // f32 of a row of a 64 x 64 matrix in LDS (rows on 16 bytes, in different banks)

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// c += A B of 16 x 16 blocks in LDS, f32.
__device__ __forceinline__ f32x4 block_product(const float* A, const float* B, f32x4 c) {
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int k = 0; k < 4; k++) c = mfma_f32(A[r * kPitch + 4 * k + g], B[(4 * k + g) * kPitch + r], c);
    return c;
}
__device__ __forceinline__ void block_store(float* D, f32x4 v, float sign) {
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; i++) D[(4 * g + i) * kPitch + r] = sign * v[i];
}

// ---- what does not depend on the state

// LDS: K's terms while products of q and k are made, then two 64 x 64 matrices in their place; what belongs to rows behind them.
template <int DKP, int NT> struct ChunkLds {
    static constexpr uint32_t kMatrix = kChunk * kPitch * 4, kRows = Layout<DKP, NT>::kOp > 2 * kMatrix ? Layout<DKP, NT>::kOp : 2 * kMatrix;
    static constexpr uint32_t kBytes = kRows + 4 * kChunk * 12 + 2 * kChunk * 4;
};

template <int DT, int DKP, int NT> __global__ __launch_bounds__(256, DKP * NT <= 256 ? 4 : 2) void delta_chunk_kernel(ChunkArgs a) {
    using L = Layout<DKP, NT>;
    using C = ChunkLds<DKP, NT>;
    constexpr int KS = DKP / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    u32x4* kop = (u32x4*)lds;                                   // [NT][4][KS][64]
    float* Am = (float*)lds;                                     // [64][kPitch]: A, and block by block T in its place
    float* Mm = Am + kChunk * kPitch;                            // P, then products on the way to T
    double* sums = (double*)(lds + C::kRows);                    // [4][64]: of four heads
    float* bt = (float*)(sums + 4 * kChunk);                     // [4][64]
    float* rk = bt + 4 * kChunk;                                 // [64]
    float* rq = rk + kChunk;
    const DeltaArgs& d = a.d;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15u, g = lane >> 4;
    const uint32_t units = d.hk * a.parts, slot = a.lo + blockIdx.x / units, kh = blockIdx.x % units / a.parts, part = blockIdx.x % a.parts;
    const uint32_t seq = seq_of(a, slot);
    const DeltaSeq s = delta_seq(d, seq);
    const uint32_t first = first_slot(s.from, seq, a.by_tokens);
    if (!s.any || slot < first || s.to - s.from <= kFewTokens || (uint64_t)(slot - first) * kChunk >= s.to - s.from) return;
    const uint32_t t0 = s.from + (slot - first) * kChunk, n = s.to - t0 < kChunk ? s.to - t0 : kChunk;
    uint8_t* out = a.scratch + (size_t)(slot - a.lo) * L::slot_bytes(d.hk, d.hv);
    uint8_t* key_out = out + (size_t)kh * L::kKeyBytes;
    const uint32_t t = 16 * wave + r;                            // this lane's row of K and Q
    // its value heads: all that share the key head, or one of them
    const uint32_t all = d.hv / d.hk, group = a.parts > 1 ? part + 1 : all, x0 = a.parts > 1 ? part : 0;
    float gt = 0.f, beta = 0.f;                                  // of a token of one of the first four heads
    auto load_decay = [&](uint32_t x) {
        gt = beta = 0.f;
        if (lane < n && x + wave < group) {
            gt = d.g[(size_t)(t0 + lane) * d.hv + kh * all + x + wave];
            beta = d.beta[(size_t)(t0 + lane) * d.hv + kh * all + x + wave];
        }
    };
    load_decay(x0);
    u32x4 kf[KS][NT], qf[KS][NT];
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        float v[8] = {};
        const uint32_t c = 32 * ks + 8 * g;
        if (t < n) load8<DT>(d.k, (size_t)(t0 + t) * d.k_stride + (size_t)kh * d.dk, c, d.dk, a.whole, v);
#pragma unroll
        for (int j = 0; j < 8; j++) kk += v[j] * v[j];
        terms8<NT>(v, kf[ks]);
        float w[8] = {};
        if (t < n) load8<DT>(d.q, (size_t)(t0 + t) * d.q_stride + (size_t)kh * d.dk, c, d.dk, a.whole, w);
#pragma unroll
        for (int j = 0; j < 8; j++) qq += w[j] * w[j];
        terms8<NT>(w, qf[ks]);
    }
    kk += __shfl_xor(kk, 16, 64);
    kk += __shfl_xor(kk, 32, 64);
    qq += __shfl_xor(qq, 16, 64);
    qq += __shfl_xor(qq, 32, 64);
    if (g == 0) {
        const bool norm = d.norm_eps >= 0.f;
        // (sums of squares past f32's range: 0 * inf would be in A and P where token by token there are zeros, so the walk is told)
        rk[t] = t >= n ? 0.f : !(kk + qq < INFINITY) ? NAN : norm ? 1.f / sqrtf(kk + d.norm_eps) : 1.f;
        rq[t] = t >= n ? 0.f : norm ? d.scale / sqrtf(qq + d.norm_eps) : d.scale;
    }
#pragma unroll
    for (int p = 0; p < NT; p++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const uint32_t at = ((p * 4 + wave) * KS + ks) * 64 + lane;
            kop[at] = kf[ks][p];
            if (part == 0) {
                ((u32x4*)key_out)[at] = kf[ks][p];
                ((u32x4*)(key_out + L::kOp))[at] = qf[ks][p];
            }
        }
    __syncthreads();
    // K^T: row d of 16 dt + r, tokens 32 ts + 8 g + e
    for (uint32_t u = part ? NT * (DKP / 16) * 2 : wave; u < NT * (DKP / 16) * 2; u += 4) {
        const uint32_t p = u / ((DKP / 16) * 2), dt = u / 2 % (DKP / 16), ts = u & 1u, dd = 16 * dt + r;
        const uint16_t* from = (const uint16_t*)kop + (size_t)p * kChunk * DKP + ((dd >> 5) * 64 + ((dd >> 3) & 3u) * 16) * 8 + (dd & 7u);
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t h[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t tt = 32 * ts + 8 * g + 2 * j + e;
                h[e] = from[((tt >> 4) * KS * 64 + (tt & 15u)) * 8];
            }
            v[j] = h[0] | h[1] << 16;
        }
        ((u32x4*)(key_out + 2 * L::kOp))[u * 64 + lane] = v;
    }
    // k_t . k_s and q_t . k_s of rows 16 wave .. and the blocks of columns up to the diagonal
    f32x4 G[4] = {}, H[4] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (j <= (int)wave)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            u32x4 b[NT];
#pragma unroll
            for (int p = 0; p < NT; p++) b[p] = kop[((p * 4 + j) * KS + ks) * 64 + lane];
            G[j] = mfma_terms(kf[ks], b, G[j]);
            H[j] = mfma_terms(qf[ks], b, H[j]);
        }
    }
    for (uint32_t x = x0; x < group; x++) {
        const uint32_t h = kh * all + x, of = (x - x0) % 4;
        uint8_t* head_out = out + (size_t)d.hk * L::kKeyBytes + (size_t)h * kHeadBytes;
        __syncthreads();   // (K's terms, and the head before: no longer read)
        if (of == 0 && x + wave < group) {   // four heads' decays and betas, one to a wave
            if (x != x0) load_decay(x);
            // (e^-100000 is 0, and a sum with -inf would have no differences)
            double sum = gt < -1e5f ? -1e5 : (double)gt;
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(sum, o, 64);
                if ((int)lane >= o) sum += up;
            }
            sums[wave * 64 + lane] = sum;
            bt[wave * 64 + lane] = beta;
            const double last = __shfl(sum, 63, 64);
            float* sc = (float*)(head_out + (size_t)wave * kHeadBytes + 2 * kTriBytes);
            const float e = __expf((float)sum);
            const float later = __expf((float)(last - sum));
            sc[lane] = beta * later * 0.f == 0.f ? e * rk[lane] : NAN;   // (what is no number would meet zeros in T and W, too: the walk is told here)
            sc[64 + lane] = e * rq[lane];
            sc[128 + lane] = rk[lane] * later;
            sc[192 + lane] = __expf((float)last);
        }
        if (of == 0) __syncthreads();
        const double* sm = sums + of * 64;
        const float* bx = bt + of * 64;
        double rs64[4];
        float rbeta[4], rqs[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = 16 * wave + 4 * g + i;
            rs64[i] = sm[row];
            rbeta[i] = bx[row] * rk[row];
            rqs[i] = rq[row];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t col = 16 * j + r;
            if (j > (int)wave) {   // (of the blocks above the diagonal (0, 1) and (2, 3) are read)
                if (j == (int)(wave ^ 1u))
#pragma unroll
                    for (int i = 0; i < 4; i++) Am[(16 * wave + 4 * g + i) * kPitch + col] = Mm[(16 * wave + 4 * g + i) * kPitch + col] = 0.f;
                continue;
            }
            const double cs = sm[col];
            const float rs = rk[col];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t row = 16 * wave + 4 * g + i;
                const float f = rs * __expf((float)(rs64[i] - cs));   // (off by 2^-24 times its exponent: at most 2^-25 of 1)
                float pv = rqs[i] * f * H[j][i], av = rbeta[i] * f * G[j][i];
                if (j == (int)wave) {
                    if (col > row) pv = 0.f;
                    if (col >= row) av = 0.f;
                }
                Am[row * kPitch + col] = av;
                Mm[row * kPitch + col] = pv;
            }
        }
        __syncthreads();
        auto put = [&](const float* M, uint8_t* to, bool by_beta) {   // rows 16 wave .. of M in terms, the steps of the triangle
            const uint32_t steps = wave < 2 ? 1 : 2, at = wave < 2 ? wave : 2 * wave - 2;
            for (uint32_t ks = 0; ks < steps; ks++) {
                const uint32_t c = 32 * ks + 8 * g;
                float v[8];
                const float4 lo = *(const float4*)(M + t * kPitch + c), hi = *(const float4*)(M + t * kPitch + c + 4);
                v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
                if (by_beta)
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] *= bx[c + e];
                u32x4 w[3];
                terms8<3>(v, w);
#pragma unroll
                for (int p = 0; p < 3; p++) ((u32x4*)to)[((at + ks) * 3 + p) * 64 + lane] = w[p];
            }
        };
        put(Mm, head_out + kTriBytes, false);
        {   // the block on the diagonal: each lane a column of its inverse (four lanes the same one), row by row
            float* D = Am + 16 * wave * (kPitch + 1);
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float sum = i == (int)r ? 1.f : 0.f;
#pragma unroll
                for (int k = 0; k < i; k++) sum -= D[i * kPitch + k] * v[k];
                v[i] = sum;
            }
            if (g == 0)
#pragma unroll
                for (int i = 0; i < 16; i++) D[i * kPitch + r] = v[i];
        }
        __syncthreads();
        auto at = [&](float* M, int i, int j) { return M + 16 * (i * kPitch + j); };
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        // pairs of blocks: (1, 0) by wave 0, (3, 2) by wave 2
        const int b = (int)wave;
        if ((b & 1) == 0) {
            block_store(at(Mm, b + 1, b), block_product(at(Am, b + 1, b), at(Am, b, b), zero), 1.f);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            block_store(at(Am, b + 1, b), block_product(at(Am, b + 1, b + 1), at(Mm, b + 1, b), zero), -1.f);
        }
        __syncthreads();
        // the lower left quarter: wave 2 i + j its block (2 + i, j)
        const int i = b >> 1, j = b & 1;
        f32x4 m = block_product(at(Am, 2 + i, 1), at(Am, 1, j), zero);   // (block (0, 1) is zero)
        m = block_product(at(Am, 2 + i, 0), at(Am, 0, j), m);
        block_store(at(Mm, 2 + i, j), m, 1.f);
        __syncthreads();
        m = block_product(at(Am, 2 + i, 2), at(Mm, 2, j), zero);
        if (i) m = block_product(at(Am, 3, 3), at(Mm, 3, j), m);
        block_store(at(Am, 2 + i, j), m, -1.f);
        __syncthreads();
        put(Am, head_out, true);
    }
}

// ---- the walk

// LDS is all that a workgroup's waves exchange: loads on their way to registers are not waited for.
__device__ __forceinline__ void walk_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Rows of N 16-bit values, one for each of 16 columns, read 16 bytes a lane at the same place of all columns, and written 8 bytes a lane: the
// 16-byte pieces of column r lie in an order turned by r, so that the sixteen columns' are in different banks.
template <int N> struct Columns {
    uint16_t v[16][N];
    static constexpr int PLANE = 16 * N;
    __device__ __forceinline__ uint16_t* at(uint32_t r, uint32_t i) {
        constexpr uint32_t PIECES = N / 8;
        const uint32_t turn = PIECES >= 16 ? r : r >> 1;   // (rows of 128 bytes lie two and two in the banks' 256)
        return &v[0][0] + r * N + (((i >> 3) ^ turn) & (PIECES - 1)) * 8 + (i & 7u);
    }
};

template <int DKP> struct WalkLds {
    Columns<DKP> S[3];                             // terms of the state
    Columns<kChunk> X[3], U[3], W[3];
    uint32_t touched[64];                          // where the words that bring lines into the L2 end up
    uint32_t bad;                                  // a chunk's U has an infinity or a NaN, or is next to one
};

struct WalkPlace {
    const uint8_t* base;     // the first chunk's slot
    size_t slot_bytes;
    uint32_t begin, end;     // chunks
    uint32_t from, to;       // tokens
    uint32_t h, kh, c0;
    size_t state;            // element of the states where this head's are
    const float* state_from;
};

// Half of the waves (AHEAD) have K S0 and U, the others Q S0 and P U, each of 16 rows; all have a share of the state's rows. Each role has a loop
// of its own, so that each wave waits for just what it loaded: what a chunk needs is asked for in the step after the one that has used the same
// registers, behind that step's reads of LDS. Between the barriers of a chunk (a, b, c):
//   a..b: X = V - e^G r (K S0)         | Y = Q S0 + P U of the chunk before, to memory
//   b..c: U = T X                      | Q S0
//   c..a: S1 = e^G S0 + K^T (r e^.. U), its terms to LDS
//
// A product with a triangle multiplies what is behind a token by zero, which an infinity or a NaN there survives, and so does the inverse of one
// whose updates leave f32's range: a chunk with such a number in U (all of X and T that is no number comes out there) is left, with the tokens
// behind it, to the token by token form, and the state before it to state_out. Returns that chunk, or w.end.
template <int DT, int DKP, int NT, bool AHEAD> __device__ __forceinline__ uint32_t walk(const DeltaArgs& d, const WalkPlace& w, WalkLds<DKP>& lds, uint32_t wave) {
    using L = Layout<DKP, NT>;
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    constexpr int KS = DKP / 32, TILES = DKP / 16, NS = TILES > 8 ? TILES / 8 : 1;   // NS: 16-row tiles of the state a wave has
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t mine = wave & 3u;
    const bool long_row = mine >= 2;                                       // two steps of a triangle
    const bool has_state = wave * NS < TILES;
    const uint32_t tile0 = has_state ? wave * NS : 0;
    const uint32_t col = w.c0 + r;
    const bool col_in = col < d.dv;
    f32x4 S[NS] = {};
    const size_t state = w.state + (size_t)(col_in ? col : 0) * d.dk;
    if (w.state_from && col_in && has_state)
#pragma unroll
        for (int x = 0; x < NS; x++) {
            const uint32_t row = 16 * (tile0 + x) + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (row + i < d.dk) S[x][i] = w.state_from[state + row + i];
        }
    u32x4 mf[KS][NT], tf[2][3], kt[NS][2][NT];
    f32x4 e, wk = {};
    float keep;
    uint32_t v[4] = {};
    // Operands of a slot lie 16 bytes a lane; what differs between loads is the same for all lanes and goes into the scalar offset.
    const uint32_t head_at = d.hk * L::kKeyBytes + w.h * kHeadBytes, rows_at = w.kh * L::kKeyBytes + (AHEAD ? 0 : L::kOp);
    const uint32_t tri_at = head_at + (AHEAD ? 0 : kTriBytes), kt_at = w.kh * L::kKeyBytes + 2 * L::kOp + tile0 * 2048, scal_at = head_at + 2 * kTriBytes;
    auto get = [&](__amdgpu_buffer_rsrc_t slot, uint32_t at) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(slot, lane * 16, at, 0)); };
    auto slot = [&](uint32_t chunk) { return kr_rsrc((uint64_t)(uintptr_t)(w.base + (size_t)(chunk - w.begin) * w.slot_bytes), (uint32_t)w.slot_bytes); };
    auto four = [&](__amdgpu_buffer_rsrc_t s, uint32_t at) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(s, g * 16, at, 0)); };
    auto load_rows = [&](__amdgpu_buffer_rsrc_t s) {        // K's or Q's rows, and the factors of their products with the state
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int k = 0; k < NT; k++) mf[ks][k] = get(s, rows_at + ((k * 4 + mine) * KS + ks) * 1024);
        e = four(s, scal_at + (AHEAD ? 0 : 256) + 64 * mine);
    };
    auto load_tri = [&](__amdgpu_buffer_rsrc_t s) {         // T's or P's (a row without a second step: nothing is read there)
        uint32_t none = long_row ? 0 : KR_OOB;
        asm volatile("" : "+s"(none));                      // (added anew: a register less)
        const uint32_t second = lane * 16 + none;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t step = (mine < 2 ? mine : 2 * mine - 2) + (j && long_row ? 1 : 0);
#pragma unroll
            for (int k = 0; k < 3; k++) tf[j][k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(s, j ? second : lane * 16, tri_at + (step * 3 + k) * 1024, 0));
        }
        if (AHEAD) wk = four(s, scal_at + 512 + 64 * mine);
    };
    auto load_kt = [&](__amdgpu_buffer_rsrc_t s) {
#pragma unroll
        for (int x = 0; x < NS; x++)
#pragma unroll
            for (int ts = 0; ts < 2; ts++)
#pragma unroll
                for (int k = 0; k < NT; k++) kt[x][ts][k] = get(s, kt_at + ((k * TILES + x) * 2 + ts) * 1024);
        keep = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(s, 0, scal_at + 768, 0));
    };
    uint32_t v_at[4];                                       // a chunk's rows of v; rows behind the sequence are behind its buffer, and read as zeros
#pragma unroll
    for (int i = 0; i < 4; i++) v_at[i] = col_in ? ((16 * mine + 4 * g + i) * (uint32_t)d.v_stride + w.h * d.dv + col) * ES : KR_OOB;
    auto load_v = [&](uint32_t chunk) {
        const uint32_t t0 = w.from + chunk * kChunk, n = t0 >= w.to ? 0 : w.to - t0 < kChunk ? w.to - t0 : kChunk;
        const uint32_t bytes = n ? ((n - 1) * (uint32_t)d.v_stride + d.hv * d.dv) * ES : 0;
        const __amdgpu_buffer_rsrc_t s = kr_rsrc((uint64_t)(uintptr_t)d.v + (uint64_t)(n ? t0 : w.from) * d.v_stride * ES, bytes);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == DT_F32) v[i] = __builtin_amdgcn_raw_buffer_load_b32(s, v_at[i], 0, 0);
            else v[i] = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(s, v_at[i], 0, 0);
        }
    };
    auto value = [&](uint32_t x) { return DT == DT_F32 ? __uint_as_float(x) : DT == DT_BF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x); };
    auto put = [&](uint16_t* to, uint32_t plane, const f32x4& x) {   // four rows of a column, in terms
        uint32_t w0[3], w1[3];
        terms<3>(x[0], x[1], w0);
        terms<3>(x[2], x[3], w1);
#pragma unroll
        for (int k = 0; k < 3; k++) *(uint2*)(to + k * plane) = make_uint2(w0[k], w1[k]);
    };
    auto put_state = [&]() {
        if (has_state)
#pragma unroll
            for (int x = 0; x < NS; x++) put(lds.S[0].at(r, 16 * (tile0 + x) + 4 * g), Columns<DKP>::PLANE, S[x]);
    };
    // `load` is what is asked for once the LDS reads are on their way.
    auto times_state = [&](f32x4& c, auto&& load) {
        constexpr int AT_ONCE = KS < 4 ? KS : 4;
        f32x4 part[4] = {};
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += AT_ONCE) {
            u32x4 b[AT_ONCE][3];
#pragma unroll
            for (int ks = 0; ks < AT_ONCE; ks++)
#pragma unroll
                for (int k = 0; k < 3; k++) b[ks][k] = *(const u32x4*)lds.S[k].at(r, 32 * (k0 + ks) + 8 * g);
            __builtin_amdgcn_sched_barrier(0);
            if (k0 == 0) load();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < AT_ONCE; ks++) mfma_terms_on(mf[k0 + ks], b[ks], part, 0);
        }
        c = (part[0] + part[1]) + (part[2] + part[3]);
    };
    auto triangle = [&](Columns<kChunk>* B, f32x4& c, auto&& load) {
        u32x4 b[2][3];
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
            for (int k = 0; k < 3; k++) b[ks][k] = *(const u32x4*)B[k].at(r, 32 * ks + 8 * g);
        __builtin_amdgcn_sched_barrier(0);
        load();
        __builtin_amdgcn_sched_barrier(0);
        f32x4 part[3] = {c};
        mfma_terms_on(tf[0], b[0], part, 0);
        if (long_row) mfma_terms_on(tf[1], b[1], part, 0);
        c = part[0] + part[1] + part[2];
    };
    f32x4 y = {};
    const uint32_t y_at = (4 * g * d.hv * d.dv + w.h * d.dv + col) * 4;
    auto give_y = [&](uint32_t chunk, auto&& load) {  // P U of a chunk onto its Q S0
        triangle(lds.U, y, load);
        const uint32_t t0 = w.from + chunk * kChunk, n = w.to - t0 < kChunk ? w.to - t0 : kChunk, row = d.hv * d.dv * 4;
        const __amdgpu_buffer_rsrc_t s = kr_rsrc((uint64_t)(uintptr_t)d.y + (uint64_t)t0 * row, n * row);   // (rows behind the sequence are not written)
#pragma unroll
        for (int i = 0; i < 4; i++) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[i]), s, col_in ? y_at + (16 * mine + i) * row : KR_OOB, 0, 0);
    };
    auto nothing = [] {};
    {
        const auto s = slot(w.begin);
        load_rows(s);
        if (AHEAD) { load_tri(s); load_v(w.begin); }
    }
    put_state();
    if (AHEAD) __builtin_amdgcn_s_setprio(3);
    uint32_t c = w.begin;
    for (; c < w.end; c++) {
        const auto here = slot(c), next = slot(c + 1 < w.end ? c + 1 : c);
        walk_barrier();
        if constexpr (AHEAD) {
            f32x4 x;
            times_state(x, [&] { load_kt(here); });
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = value(v[i]) - e[i] * x[i];
            asm volatile("" : "+v"(x));   // (here, not behind the next loads into e's and v's registers)
            put(lds.X[0].at(r, 16 * mine + 4 * g), Columns<kChunk>::PLANE, x);
        } else if (c > w.begin) {
            give_y(c - 1, [&] { load_kt(here); });
        } else {
            load_kt(here);
        }
        walk_barrier();
        f32x4 late;
        if constexpr (AHEAD) {
            f32x4 u = {};
            triangle(lds.X, u, [&] { load_rows(next); load_v(c + 1); });
            f32x4 uw = u * wk;
            asm volatile("" : "+v"(uw));
            put(lds.W[0].at(r, 16 * mine + 4 * g), Columns<kChunk>::PLANE, uw);
            // (magnitudes whose terms could round to infinities count, too: a term of 3.39e38 and more would)
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) most += fabsf(u[i]) + fabsf(uw[i]);
            if (__ballot(!(most < 3.3e38f))) lds.bad = 1;
            late = u;   // (U itself is asked for from the next chunk on: it is put beside the state's update)
        } else {
            times_state(y, [&] { load_tri(here); });
            y *= e;
            asm volatile("" : "+v"(y));
        }
        walk_barrier();
        const uint32_t bad = lds.bad;
        u32x4 b[2][3];
#pragma unroll
        for (int ts = 0; ts < 2; ts++)
#pragma unroll
            for (int k = 0; k < 3; k++) b[ts][k] = *(const u32x4*)lds.W[k].at(r, 32 * ts + 8 * g);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (AHEAD) {
            load_tri(next);
            put(lds.U[0].at(r, 16 * mine + 4 * g), Columns<kChunk>::PLANE, late);
        } else {
            load_rows(next);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_amdgcn_readfirstlane(bad)) break;
        if (has_state) {
#pragma unroll
            for (int x = 0; x < NS; x++) {
                f32x4 part[2] = {S[x] * keep, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int ts = 0; ts < 2; ts++) mfma_terms_on(kt[x][ts], b[ts], part, ts);
                S[x] = part[0] + part[1];
            }
        }
        put_state();
    }
    if (AHEAD) __builtin_amdgcn_s_setprio(0);
    if (c == w.end) {
        walk_barrier();   // (the last chunk's U)
        if constexpr (!AHEAD) give_y(w.end - 1, nothing);
    }
    if (col_in && has_state)
#pragma unroll
        for (int x = 0; x < NS; x++) {
            const uint32_t row = 16 * (tile0 + x) + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (row + i < d.dk) d.state_out[state + row + i] = S[x][i];
        }
    return c;
}

// The walk's last wave: brings what the others read kAheadChunks chunks later from memory into the XCD's L2, a word of every 128-byte line (a
// chunk takes less time than a line's way from memory, and registers hold one chunk ahead). The words go to LDS, so that nothing waits for
// them. The workgroups of a head's columns share its lines. (M0 is read one wait state behind its write at the earliest.)
constexpr uint32_t kAheadChunks = 4;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // M0 is a reserved register: naming it as clobbered is the point
__device__ __forceinline__ void touch(const void* line, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(line) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int DT, int DKP, int NT> __device__ __forceinline__ void walk_touch(const DeltaArgs& d, const WalkPlace& w, WalkLds<DKP>& lds, uint32_t columns) {
    using L = Layout<DKP, NT>;
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint32_t*)lds.touched);
    const uint32_t key_at = w.kh * L::kKeyBytes, head_at = d.hk * L::kKeyBytes + w.h * kHeadBytes;
    constexpr uint32_t KEY_LINES = L::kKeyBytes / 128, LINES = KEY_LINES + kHeadBytes / 128;
    auto chunk = [&](uint32_t c) {
        const uint8_t* p = w.base + (size_t)(c - w.begin) * w.slot_bytes;
        for (uint32_t i0 = w.c0 / 16 * 64; i0 < LINES; i0 += 64 * columns) {
            const uint32_t i = i0 + lane < LINES ? i0 + lane : LINES - 1;
            touch(p + (i < KEY_LINES ? key_at + i * 128 : head_at + (i - KEY_LINES) * 128), to);
        }
        const uint32_t t = w.from + c * kChunk + lane;
        // (the whole word that holds the row's first element: nothing past the last page of v)
        touch((const uint8_t*)(((uintptr_t)d.v + ((size_t)(t < w.to ? t : w.to - 1) * d.v_stride + (size_t)w.h * d.dv + w.c0) * ES) & ~(uintptr_t)3), to);
    };
    for (uint32_t c = w.begin; c < w.end && c < w.begin + kAheadChunks; c++) chunk(c);
    for (uint32_t c = w.begin; c < w.end; c++) {
        if (c + kAheadChunks < w.end) chunk(c + kAheadChunks);
        walk_barrier();
        walk_barrier();
        walk_barrier();
        if (__builtin_amdgcn_readfirstlane(lds.bad)) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            return;
        }
    }
    walk_barrier();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int DT, int DKP, int NT, bool TOUCH, int PER_SIMD> __global__ __launch_bounds__(64 * (8 + TOUCH), PER_SIMD) void delta_walk_kernel(ChunkArgs a, uint32_t pairs, uint32_t beside, uint32_t columns) {
    using L = Layout<DKP, NT>;
    __shared__ __attribute__((aligned(16))) WalkLds<DKP> lds;
    const DeltaArgs& d = a.d;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go to the eight XCDs in turn: the column blocks of a head, and of `beside` heads side by side, to one, whose L2 then has what they
    // share; the heads of a sequence, which end together, to as many XCDs as there are.
    const uint32_t i = blockIdx.x / 8, pair = (i / (beside * columns) * 8 + blockIdx.x % 8) * beside + i / columns % beside, c0 = i % columns * 16;
    if (pair >= pairs) return;
    const uint32_t seq = pair / d.hv, h = pair % d.hv;
    const DeltaSeq s = delta_seq(d, seq);
    if (!s.any) return;
    const uint32_t len = s.to - s.from, first = first_slot(s.from, seq, a.by_tokens);
    DeltaSeq one = s;                      // what goes token by token, and from which states
    const float* from = d.state_in;
    if (len <= kFewTokens) {
        if (first < a.lo || first >= a.hi) return;
    } else {
        const uint32_t chunks = (len + kChunk - 1) / kChunk;
        WalkPlace w;
        w.begin = a.lo > first ? a.lo - first : 0;
        w.end = a.hi <= first ? 0 : a.hi - first < chunks ? a.hi - first : chunks;
        if (w.begin >= w.end) return;
        w.slot_bytes = L::slot_bytes(d.hk, d.hv);
        w.base = a.scratch + (size_t)(first + w.begin - a.lo) * w.slot_bytes;
        w.from = s.from;
        w.to = s.to;
        w.h = h;
        w.kh = h / (d.hv / d.hk);
        w.c0 = c0;
        w.state = ((size_t)s.slot * d.hv + h) * d.dv * d.dk;
        w.state_from = w.begin ? d.state_out : d.state_in;
        if (threadIdx.x == 0) lds.bad = 0;
        uint32_t done;
        if (wave < 4) {
            done = walk<DT, DKP, NT, true>(d, w, lds, wave);
        } else if (wave < 8) {
            done = walk<DT, DKP, NT, false>(d, w, lds, wave);
        } else {
            if constexpr (TOUCH) walk_touch<DT, DKP, NT>(d, w, lds, columns);
            return;
        }
        if (done == w.end) return;
        __syncthreads();                   // (the states are in memory)
        one.from = s.from + done * kChunk;
        if (w.end < chunks) one.to = s.from + w.end * kChunk;
        from = d.state_out;
    }
    if (wave >= 4) return;
    DeltaArgs tokens = d;
    tokens.state_in = from;
    if (a.whole && d.dk == DKP) delta_tokens<DT, DKP / 16, true>(tokens, one, h, c0 + 4 * wave);
    else delta_tokens<DT, DKP / 16, false>(tokens, one, h, c0 + 4 * wave);
}

// Heads that share a key head go to one XCD where that leaves none without (nine prompts of 1 to 1024 tokens, f16: 75 -> 53 us in both launches
// against runs of heads, the long prompt's all on one).
uint32_t heads_beside(const DeltaArgs& d) { return (uint64_t)d.n_seqs * d.hk >= 8 ? d.hv / d.hk : 1; }
uint64_t walk_grid(const DeltaArgs& d) {
    const uint32_t beside = heads_beside(d);
    return ((uint64_t)d.n_seqs * d.hv / beside + 7) / 8 * 8 * beside * ((d.dv + 15) / 16);
}

template <int DT, int DKP, int NT> int launch_chunks(const DeltaArgs& d, void* scratch, size_t bytes, const LaunchCtx& lc) {
    using L = Layout<DKP, NT>;
    ChunkArgs a;
    a.d = d;
    a.scratch = (uint8_t*)scratch;
    a.whole = delta_rows_whole(d);
    const uint32_t total = (uint32_t)slots_of(d, a.by_tokens), at_once = (uint32_t)(bytes / L::slot_bytes(d.hk, d.hv));
    uint32_t pairs = d.n_seqs * d.hv, columns = (d.dv + 15) / 16, beside = heads_beside(d);
    const uint64_t grid = walk_grid(d);   // (the first launch has less than 2^16 workgroups, as a slot of the scratch has more than 16 KB a head)
    // A wave more makes three on one of the four SIMDs, 168 registers each: rows of 384 terms and more need up to 256, and go without. Two
    // workgroups to a compute unit need 128: rows of 64 bf16 or f16 values do with them, and where there are more workgroups than compute units
    // that gives more than the lines brought early (nine prompts of 1 to 1024 tokens, f16: 54 us against 64 with the wave and 60 without either).
    // Four prompts of 2048 tokens, dk 128: bf16 298 us with the wave, 346 without; f16 376, 459; f32 878 (its registers do not fit), 563.
    constexpr bool wide = DKP * NT >= 384, narrow = DKP == 64 && NT <= 2;
    const bool touch = !wide && !(narrow && grid > 256);
    const void* fn;
    if constexpr (wide) fn = (const void*)delta_walk_kernel<DT, DKP, NT, false, 2>;
    else if constexpr (narrow) fn = touch ? (const void*)delta_walk_kernel<DT, DKP, NT, true, 1> : (const void*)delta_walk_kernel<DT, DKP, NT, false, 4>;
    else fn = (const void*)delta_walk_kernel<DT, DKP, NT, true, 1>;
    constexpr size_t lds = ChunkLds<DKP, NT>::kBytes;
    const void* chunk = (const void*)delta_chunk_kernel<DT, DKP, NT>;
    MTQ_HIP(set_max_dynamic_lds(chunk, lds));
    for (uint32_t lo = 0; lo < total; lo += at_once) {
        a.lo = lo;
        a.hi = total - lo < at_once ? total : lo + at_once;
        LaunchCtx first = lc, second = lc;
        first.stop = nullptr;
        if (lo) first.start = nullptr;
        second.start = nullptr;
        if (a.hi < total) second.stop = nullptr;
        void* args[] = {&a, &pairs, &beside, &columns};
        // Few chunks: a workgroup for each value head, which all work out the products of q and k that they share.
        a.parts = (uint64_t)(a.hi - lo) * d.hk < 512 ? d.hv / d.hk : 1;
        MTQ_HIP(launch_kernel(chunk, dim3((a.hi - lo) * d.hk * a.parts), dim3(256), args, lds, first));
        MTQ_HIP(launch_kernel(fn, dim3((uint32_t)grid), dim3(64 * (8 + touch)), args, 0, second));
    }
    return ERR_OK;
}

template <int DT, int NT> int pick(const DeltaArgs& d, void* scratch, size_t bytes, const LaunchCtx& lc) {
    return d.dk <= 64 ? launch_chunks<DT, 64, NT>(d, scratch, bytes, lc) : d.dk <= 128 ? launch_chunks<DT, 128, NT>(d, scratch, bytes, lc)
                                                                                        : launch_chunks<DT, 256, NT>(d, scratch, bytes, lc);
}
size_t slot_bytes_of(const DeltaArgs& d) {
    const size_t terms = d.dtype == DT_BF16 ? 1 : d.dtype == DT_F16 ? 2 : 3, dkp = d.dk <= 64 ? 64 : d.dk <= 128 ? 128 : 256;
    return d.hk * 3 * terms * kChunk * dkp * 2 + (size_t)d.hv * kHeadBytes;
}

}  // namespace

// Chunks pay where a sequence may be long: with as many tokens beyond one for each sequence as this. (Sequences of up to kFewTokens go token
// by token here too.)
// The walk reads a chunk's rows of v and a slot by 31-bit offsets, and has a workgroup for 16 columns of every head of every sequence: where these
// are more than a launch can have, sequences go token by token, all of them at once.
bool delta_chunks_serve(const DeltaArgs& d) {
    if (d.v_stride > (1u << 22) || slot_bytes_of(d) >= ((size_t)1 << 31) || walk_grid(d) > max_workgroups(64 * 9)) return false;
    return d.offsets ? d.n_tokens > d.n_seqs && d.n_tokens - d.n_seqs >= 2 * kFewTokens : d.n_tokens / d.n_seqs >= 2 * kFewTokens;
}

// All of the call's chunks at once up to a gigabyte (and what the caller allows); more go in windows, each sequence from the state that the
// window before left. 0: not even one chunk fits.
size_t delta_chunks_scratch_bytes(const DeltaArgs& d, size_t most) {
    if (most > ((size_t)1 << 30)) most = (size_t)1 << 30;
    uint32_t by_tokens;
    const size_t one = slot_bytes_of(d), all = one * slots_of(d, by_tokens);
    return all <= most ? all : most / one * one;
}

int launch_delta_chunks(const DeltaArgs& d, void* scratch, size_t bytes, const LaunchCtx& lc) {
    return d.dtype == DT_F32 ? pick<DT_F32, 3>(d, scratch, bytes, lc) : d.dtype == DT_F16 ? pick<DT_F16, 2>(d, scratch, bytes, lc) : pick<DT_BF16, 1>(d, scratch, bytes, lc);
}

}  // namespace mtq
