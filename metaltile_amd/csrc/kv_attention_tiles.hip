// Attention over the 4-bit cache for sequences of many rows (prompts): bound by the vector units beside the matrix cores.
//
// A workgroup has 64 NW.. rows of one key head (new tokens times the query heads that share it), each wave 16 MT of them as columns of its
// matrix instructions, and goes through the tokens that they see 64 at a time. Codes are made operands once for all waves: a thread turns 32 codes of keys and
// 32 of values into numbers of 16 bits on their way into the LDS, in the order in which the instructions take them, scales and biases into f32; two stages, so that
// a block's codes come from memory while the one before is computed. Four tokens of one query to a lane (kv_attention.h), so that a scale is read
// once for MT of them.
#include "kv_attention.h"

namespace mtq {

namespace {

constexpr uint32_t kBlock = 64;   // tokens

template <int DT, int D, int G, int NW> struct TilesShape {
    static constexpr int Q = KvTerms<DT>::Q, NG = D / G, STEPS = D / 32, NT = G / 16, TH = 64 * NW;
    static constexpr int MT = D * Q <= 192 ? 2 : 1;   // sixteens of rows of a wave: sums and queries fill its registers
    static constexpr int ROWS = 16 * MT * NW;
    static constexpr int VT = 1024 + 16;                          // a tile of values, and what keeps the tiles' writes in different banks
    static constexpr int K = kBlock * D * 2, V = kBlock / 32 * (D / 16) * VT, S = 4 * NG * kBlock * 4;
    static constexpr int STAGE = K + V + S;
    static constexpr int LDS = 2 * STAGE + 2 * 16 * 4;
};

template <int DT, int D, int G, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv_tiles_kernel(KvAttentionArgs a, KvParts parts, uint32_t tiles) {
    using L = TilesShape<DT, D, G, NW>;
    using T = KvTerms<DT>;
    constexpr int MT = L::MT, NG = L::NG, NT = L::NT, STEPS = L::STEPS, TH = L::TH;
    constexpr int KITEMS = (int)kBlock * (D / 32), VITEMS = (int)kBlock / 4 * (D / 8), SITEMS = 2 * (int)kBlock * NG;
    constexpr int KI = (KITEMS + TH - 1) / TH, VI = (VITEMS + TH - 1) / TH, SI = (SITEMS + TH - 1) / TH;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const KvArgs& kv = a.kv;
    const uint32_t th = threadIdx.x, lane = th & 63u, wave = __builtin_amdgcn_readfirstlane(th >> 6), r = lane & 15u, g = lane >> 4;
    const uint32_t shared = a.hq / kv.hkv, head = blockIdx.x % kv.hkv, at_slice = blockIdx.x / kv.hkv, slice = at_slice % parts.slices;
    // Sequence i's tiles begin at (its first row) * shared / ROWS + i, which leaves room for as many as it has. The last ones see the most and come first.
    const uint32_t tile = tiles - 1u - at_slice / parts.slices;
    uint32_t seq;
    if (kv.offsets) {
        uint32_t lo = 0, n = kv.n_seqs;   // of the sequences lo .. lo + n - 1 the last that begins at `tile` or before
        while (n > 1) {
            const uint32_t step = (n + 63u) / 64u, i = lo + lane * step;
            const bool before = lane * step < n && (uint32_t)((uint64_t)(kv.offsets[i] < kv.n_tokens ? kv.offsets[i] : kv.n_tokens) * shared / L::ROWS) + i <= tile;
            const uint32_t count = (uint32_t)__popcll(__ballot(before));
            const uint32_t skip = count ? (count - 1u) * step : 0u;
            lo += skip;
            n = n - skip < step ? n - skip : step;
        }
        seq = __builtin_amdgcn_readfirstlane(lo);
    } else {
        const uint64_t per = (uint64_t)(kv.n_tokens / kv.n_seqs) * shared;   // (the beginnings of equal sequences: the last i with i per / ROWS + i <= tile)
        uint32_t i = (uint32_t)((uint64_t)tile * L::ROWS / (per + L::ROWS));
        while (i + 1u < kv.n_seqs && (i + 1u) * per / L::ROWS + i + 1u <= tile) i++;
        seq = i;
    }
    const KvSeq s = kv_seq(kv, seq);
    const uint32_t rows = s.rows * shared, first_tile = (uint32_t)((uint64_t)s.first_row * shared / L::ROWS) + seq;
    if (tile < first_tile || (uint64_t)(tile - first_tile) * L::ROWS >= rows) return;
    const uint32_t row0 = (tile - first_tile) * L::ROWS;

    auto end_of = [&](uint32_t i) { const int32_t e = (int32_t)(s.len + i / shared + 1u) - (int32_t)s.rows; return e > 0 ? (uint32_t)e : 0u; };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    const uint32_t last = row0 + L::ROWS - 1u < rows ? row0 + L::ROWS - 1u : rows - 1u;
    const uint32_t hi = __builtin_amdgcn_readfirstlane(end_of(last)), lo = __builtin_amdgcn_readfirstlane(from_of(end_of(row0))) & ~31u;
    const uint32_t blocks = kv.n_pages && hi > lo ? (hi - lo + kBlock - 1u) / kBlock : 0u, per = (blocks + parts.slices - 1u) / parts.slices;
    const uint32_t b0 = slice * per < blocks ? slice * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
    // This wave's rows, and a lane's.
    const uint32_t wave0 = row0 + wave * 16 * MT, wave_last = wave0 + 16 * MT - 1u < rows ? wave0 + 16 * MT - 1u : rows - 1u;
    const bool any = wave0 < rows;
    const uint32_t first_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave0) : 0u), last_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave_last) : 0u);
    const uint32_t first_from = from_of(first_end), last_from = from_of(last_end);
    uint32_t end[MT], from[MT];
    uint64_t row_at[MT];   // its row of the call
    uint32_t qh[MT];
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);   // (not 0: what is hidden scores -inf)
    kr_u32x4 q[MT][T::Q][STEPS];
    float qsum[MT][NG] = {};
#pragma unroll
    for (int m = 0; m < MT; m++) {
        uint32_t i = wave0 + 16 * m + r;
        if (i >= rows) i = rows - 1u;
        end[m] = end_of(i);
        from[m] = from_of(end[m]);
        row_at[m] = s.first_row + i / shared;
        qh[m] = head * shared + i % shared;
        const uint64_t q_at = row_at[m] * a.q_stride + (uint64_t)qh[m] * D + 8 * g;
#pragma unroll
        for (int j0 = 0; j0 < STEPS; j0++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = load_elem<DT>(a.q, q_at + 32 * j0 + j);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] = a.scale < 0.f ? -v[j] : v[j];
                qsum[m][j0 * 32 / G] += v[j];
            }
#pragma unroll
            for (int p = 0; p < 4; p++) {
                if constexpr (DT == DT_F16) {
                    q[m][0][j0][p] = (uint32_t)f32_to_elem_bits<DT_F16>(v[p]) | (uint32_t)f32_to_elem_bits<DT_F16>(v[p + 4]) << 16;
                } else {
                    float x[T::Q], y[T::Q];
                    kv_split(v[p], x);
                    kv_split(v[p + 4], y);
#pragma unroll
                    for (int t = 0; t < T::Q; t++) q[m][t][j0][p] = kv_pack_bf16(x[t], y[t]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NG; n++) qsum[m][n] = kv_column_sum(qsum[m][n]);
    }

    // A block's codes from memory into registers, and from there as operands into its stage.
    const uint32_t k16 = kv_sixteen<T::QK>(), v16 = kv_sixteen<DT_BF16>();
    uint4 kraw[KI];
    uint32_t vraw[VI][4];
    float sraw[SI], braw[SI];
    uint32_t there = 0;   // of a block that is fetched: a bit for each of its sixteens of tokens that is on a page
    auto fetch = [&](uint32_t b) {
        const uint32_t t0 = lo + b * kBlock;
        uint64_t slot[4];
        there = 0;
#pragma unroll
        for (int h = 0; h < 4; h++) {
            const uint32_t at = t0 + 16 * h;
            const uint32_t page = at < hi ? kv.pages[(uint64_t)s.seq * kv.pages_stride + (at >> kv.page_log2)] : 0xFFFFFFFFu;
            const bool ok = page < kv.n_pages;
            there |= (uint32_t)ok << h;
            slot[h] = (((uint64_t)(ok ? page : 0u) * kv.hkv + head) << kv.page_log2) + (at & ((1u << kv.page_log2) - 1u));   // (of no page: one that is there)
        }
        auto slot_of = [&](uint32_t h) { return h & 2u ? (h & 1u ? slot[3] : slot[2]) : (h & 1u ? slot[1] : slot[0]); };
#pragma unroll
        for (int u = 0; u < KI; u++) {
            const uint32_t i = u * TH + th;
            if (KITEMS % TH == 0 || i < KITEMS)
                kraw[u] = *(const uint4*)((const uint8_t*)kv.k.codes + (slot_of(i / (16 * (D / 32))) + i % 16) * (D / 2) + i / 16 % (D / 32) * 16);
        }
#pragma unroll
        for (int u = 0; u < VI; u++) {
            const uint32_t i = u * TH + th, quad = i / (D / 8), w = i % (D / 8);
            if (VITEMS % TH == 0 || i < VITEMS) {
                const uint32_t* p = kv.v.codes + (slot_of(quad / 4) + quad % 4 * 4) * (D / 8) + w;
#pragma unroll
                for (int j = 0; j < 4; j++) vraw[u][j] = p[j * (D / 8)];
            }
        }
#pragma unroll
        for (int u = 0; u < SI; u++) {
            const uint32_t i = u * TH + th, n = i % NG, t = i / NG % kBlock;
            if (SITEMS % TH == 0 || i < SITEMS) {
                const bool value = i / (NG * kBlock);
                const void *scales = value ? kv.v.scales : kv.k.scales, *biases = value ? kv.v.biases : kv.k.biases;
                const uint64_t at = (slot_of(t / 16) + t % 16) * NG + n;
                const bool in = (there >> (t / 16) & 1u) && t0 + t < hi;   // (where no token is: zeros)
                sraw[u] = in ? load_elem<DT>(scales, at) : 0.f;
                braw[u] = in ? load_elem<DT>(biases, at) : 0.f;
            }
        }
    };
    uint32_t* const odd = (uint32_t*)(lds + 2 * L::STAGE);   // [stage][wave]: whether the values' scales or biases that the wave brought hold a NaN or an infinity
    auto store = [&](uint32_t b) {
        uint8_t* st = lds + (b & 1u) * L::STAGE;
#pragma unroll
        for (int u = 0; u < KI; u++) {
            const uint32_t i = u * TH + th;
            if (KITEMS % TH == 0 || i < KITEMS) {
                const uint32_t w[4] = {kraw[u].x, kraw[u].y, kraw[u].z, kraw[u].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    kr_u32x4 k;
#pragma unroll
                    for (int p = 0; p < 4; p++) k[p] = kv_pair<T::QK>(w[j], p, k16);
                    *(kr_u32x4*)(st + ((i / 16) * 64 + j * 16 + i % 16) * 16) = k;   // (i / 16: sixteen of tokens and step)
                }
            }
        }
#pragma unroll
        for (int u = 0; u < VI; u++) {
            const uint32_t i = u * TH + th, quad = i / (D / 8), w = i % (D / 8);
            if (VITEMS % TH == 0 || i < VITEMS) {
                uint8_t* to = st + L::K + (quad / 8 * (D / 16) + w / 2) * L::VT + (quad % 4 * 16 + w % 2 * 8) * 16 + quad / 4 % 2 * 8;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    kr_u32x2 v;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t two = __builtin_amdgcn_perm(vraw[u][2 * j + 1], vraw[u][2 * j], 0x0C000C00u | (uint32_t)(4 + e / 2) << 16 | (uint32_t)(e / 2));
                        v[j] = ((e & 1 ? two >> 1 : two << 3) & 0x00780078u) | v16;
                    }
                    *(kr_u32x2*)(to + e * 16) = v;
                }
            }
        }
        float* sc = (float*)(st + L::K + L::V);   // [K scales, K biases - 16 scales, V scales, V biases + 8 scales][group][token]
        bool fine = true;
#pragma unroll
        for (int u = 0; u < SI; u++) {
            const uint32_t i = u * TH + th, n = i % NG, t = i / NG % kBlock, value = i / (NG * kBlock);
            if (SITEMS % TH == 0 || i < SITEMS) {
                const float second = fmaf(value ? 8.f : -16.f, sraw[u], braw[u]);
                sc[((2 * value) * NG + n) * kBlock + t] = sraw[u];
                sc[((2 * value + 1) * NG + n) * kBlock + t] = second;
                fine = fine && (!value || (fabsf(sraw[u]) < INFINITY && fabsf(second) < INFINITY));
            }
        }
        const bool all_fine = __all(fine);
        if (lane == 0) odd[(b & 1u) * 16 + wave] = !all_fine;
    };

    kr_f32x4 o[MT][NG][NT] = {};
    float ones[MT][NG] = {}, bias[MT][NG] = {}, sum[MT] = {}, bar[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) bar[m] = -INFINITY;
    auto part = [&](const uint8_t* st, uint32_t sb, uint32_t t0, uint32_t on_page, uint32_t stage) {   // 32 tokens from t0 on
        const float* sc = (const float*)(st + L::K + L::V) + sb * 32 + 4 * g;
        float x[MT][2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t* kt = st + (sb * 2 + t) * (STEPS * 1024) + lane * 16;
#pragma unroll
            for (int n = 0; n < NG; n++) {
                kr_f32x4 acc[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m] = kr_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = n * (G / 32); i < (n + 1) * (G / 32); i++) {
                    const kr_u32x4 k = *(const kr_u32x4*)(kt + i * 1024);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int e = T::Q - 1; e >= 0; e--) acc[m] = kr_mfma<T::QK>(k, q[m][e][i], acc[m]);
                }
                const kr_f32x4 ks = *(const kr_f32x4*)(sc + n * kBlock + 16 * t), kb = *(const kr_f32x4*)(sc + (NG + n) * kBlock + 16 * t);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[m][t][i] = fmaf(kb[i], qsum[m][n], n ? fmaf(ks[i], acc[m][i], x[m][t][i]) : ks[i] * acc[m][i]);
            }
        }
        const bool whole = t0 >= last_from && t0 + 32u <= first_end && (on_page >> (2 * sb) & 3u) == 3u;
        uint32_t seen = 0xFFFFFFFFu;   // (8 bits for each m)
        if (!whole) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t tok = t0 + 16 * t + 4 * g + i;
                        if (!((on_page >> (2 * sb + t) & 1u) && tok >= from[m] && tok < end[m])) {
                            x[m][t][i] = -INFINITY;
                            seen &= ~(1u << (8 * m + 4 * t + i));
                        }
                    }
        }
        float top[MT];
        bool over = false;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            top[m] = fmaxf(fmaxf(fmaxf(x[m][0][0], x[m][0][1]), fmaxf(x[m][0][2], x[m][0][3])), fmaxf(fmaxf(x[m][1][0], x[m][1][1]), fmaxf(x[m][1][2], x[m][1][3])));
            over = over || top[m] * c > bar[m] + kSlack;
        }
        if (__any(over)) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const float to = fmaxf(bar[m], kv_column_max(top[m]) * c), keep = to > bar[m] ? __builtin_amdgcn_exp2f(bar[m] - to) : 1.f;
                sum[m] *= keep;
#pragma unroll
                for (int n = 0; n < NG; n++) {
                    bias[m][n] *= keep;
                    ones[m][n] *= keep;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[m][n][t][i] *= keep;
                }
                bar[m] = to;
            }
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float from_bar = bar[m] == -INFINITY ? 0.f : bar[m];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[m][t][i] = __builtin_amdgcn_exp2f(fmaf(x[m][t][i], c, -from_bar));
                    sum[m] += x[m][t][i];
                }
        }
        bool clean = true;   // (a weight of 0 does not keep a NaN out: where some rows do not see all, they are taken out, and put to the rows that see them)
        if (!whole) {
            uint32_t some = 0;
            for (int w = 0; w < NW; w++) some |= odd[stage * 16 + w];
            clean = __builtin_amdgcn_readfirstlane(some) == 0;
        }
        const kr_u32x4 less24 = {0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u};   // -24 in bf16
#pragma unroll
        for (int n = 0; n < NG; n++) {
            kr_f32x4 vs[2], vb[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                vs[t] = *(const kr_f32x4*)(sc + (2 * NG + n) * kBlock + 16 * t);
                vb[t] = *(const kr_f32x4*)(sc + (3 * NG + n) * kBlock + 16 * t);
            }
            if (!clean) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!(fabsf(vs[t][i]) < INFINITY && fabsf(vb[t][i]) < INFINITY)) {
                            vs[t][i] = vb[t][i] = 0.f;
#pragma unroll
                            for (int m = 0; m < MT; m++)
                                if (seen >> (8 * m + 4 * t + i) & 1u) bias[m][n] = __builtin_nanf("");
                        }
            }
            kr_u32x4 pt[MT][T::P];
#pragma unroll
            for (int m = 0; m < MT; m++) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) bias[m][n] = fmaf(x[m][t][i], vb[t][i], bias[m][n]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float y[2][T::P];
#pragma unroll
                    for (int e = 0; e < 2; e++) kv_split(x[m][j / 2][2 * j % 4 + e] * vs[j / 2][2 * j % 4 + e], y[e]);
#pragma unroll
                    for (int e = 0; e < T::P; e++) pt[m][e][j] = kv_pack_bf16(y[0][e], y[1][e]);
                }
                kr_f32x4 less = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = T::P - 1; e >= 0; e--) less = kr_mfma<DT_BF16>(less24, pt[m][e], less);
                ones[m][n] += less[0];
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const kr_u32x4 v = *(const kr_u32x4*)(st + L::K + (sb * (D / 16) + n * NT + t) * L::VT + lane * 16);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int e = T::P - 1; e >= 0; e--) o[m][n][t] = kr_mfma<DT_BF16>(v, pt[m][e], o[m][n][t]);
            }
        }
    };

    if (b0 < b1) {
        fetch(b0);
        uint32_t now = there, next = 0;   // (the fetched blocks' `there`)
        store(b0);
        if (b0 + 1u < b1) {
            fetch(b0 + 1u);
            next = there;
        }
        __syncthreads();
        for (uint32_t b = b0; b < b1; b++) {
            const uint32_t on_page = now;
            if (b + 1u < b1) store(b + 1u);
            now = next;
            if (b + 2u < b1) {
                fetch(b + 2u);
                next = there;
            }
            const uint32_t t0 = lo + b * kBlock;
#pragma unroll 1
            for (uint32_t sb = 0; sb < 2; sb++)
                if (t0 + 32 * sb < last_end && t0 + 32 * sb + 32u > first_from) part(lds + (b & 1u) * L::STAGE, sb, t0 + 32 * sb, on_page, b & 1u);
            __syncthreads();
        }
    }

#pragma unroll
    for (int m = 0; m < MT; m++) {
        const float total = kv_column_sum(sum[m]);
        const uint32_t i = wave0 + 16 * m + r;
        const uint64_t at = (row_at[m] * a.hq + qh[m]) * parts.slices + slice;
        if (parts.slices > 1 && i < rows && g == 0) {
            parts.sums[at * 2] = bar[m];
            parts.sums[at * 2 + 1] = total;
        }
        const float by = parts.slices > 1 ? 1.f : total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const float more = kv_column_sum(bias[m][n]) + ones[m][n];
            if (i >= rows) continue;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t d = n * G + 16 * t + 4 * g;
                kr_f32x4 v;
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = parts.slices == 1 && total == 0.f ? 0.f : (o[m][n][t][j] + more) * by;
                if (parts.slices > 1) {
                    *(kr_f32x4*)(parts.values + at * D + d) = v;
                } else {
                    const uint64_t to = row_at[m] * a.out_stride + (uint64_t)qh[m] * D + d;
                    if constexpr (DT == DT_F32)
                        *(kr_f32x4*)((float*)a.out + to) = v;
                    else
                        *(uint2*)((uint16_t*)a.out + to) = make_uint2((uint32_t)f32_to_elem_bits<DT>(v[0]) | (uint32_t)f32_to_elem_bits<DT>(v[1]) << 16,
                                                                    (uint32_t)f32_to_elem_bits<DT>(v[2]) | (uint32_t)f32_to_elem_bits<DT>(v[3]) << 16);
                }
            }
        }
    }
}

constexpr int kWaves = 4;

template <int DT, int D, int G> int launch(const KvAttentionArgs& p, KvParts parts, const LaunchCtx& lc) {
    using L = TilesShape<DT, D, G, kWaves>;
    KvAttentionArgs a = p;
    static_assert(L::LDS <= 160 * 1024, "");
    const void* fn = (const void*)kv_tiles_kernel<DT, D, G, kWaves>;
    const uint64_t tiles64 = (uint64_t)a.kv.n_tokens * (a.hq / a.kv.hkv) / L::ROWS + a.kv.n_seqs;
    if (tiles64 * a.kv.hkv * parts.slices > max_workgroups(64 * kWaves)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    uint32_t tiles = (uint32_t)tiles64;
    LaunchCtx first = lc;
    if (parts.slices > 1) first.stop = nullptr;
    MTQ_HIP(set_max_dynamic_lds(fn, L::LDS));
    void* args[] = {&a, &parts, &tiles};
    MTQ_HIP(launch_kernel(fn, dim3(tiles * a.kv.hkv * parts.slices), dim3(64 * kWaves), args, L::LDS, first));
    LaunchCtx last = lc;
    last.start = nullptr;
    return parts.slices > 1 ? launch_kv_join(DT, a, parts, last) : ERR_OK;
}

template <int DT> int launch_of(const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (p.kv.dim * 1000 + p.kv.group) {
        case 64032: return launch<DT, 64, 32>(p, parts, lc);
        case 64064: return launch<DT, 64, 64>(p, parts, lc);
        case 128032: return launch<DT, 128, 32>(p, parts, lc);
        case 128064: return launch<DT, 128, 64>(p, parts, lc);
        case 128128: return launch<DT, 128, 128>(p, parts, lc);
        case 256032: return launch<DT, 256, 32>(p, parts, lc);
        case 256064: return launch<DT, 256, 64>(p, parts, lc);
        case 256128: return launch<DT, 256, 128>(p, parts, lc);
    }
    return fail(ERR_UNSUPPORTED, "kv_attention: no kernel for this head_dim and group_size");
}

}  // namespace

int launch_kv_tiles(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (dtype) {
        case DT_F32: return launch_of<DT_F32>(p, parts, lc);
        case DT_F16: return launch_of<DT_F16>(p, parts, lc);
        default: return launch_of<DT_BF16>(p, parts, lc);
    }
}

// Rows of a tile, by which the slices are chosen.
uint32_t kv_tile_rows(int dtype, uint32_t dim) {
    const uint32_t work = dim * (dtype == DT_F32 ? 3 : 1);
    return 16 * kWaves * (work <= 192 ? 2 : 1);
}

}  // namespace mtq
