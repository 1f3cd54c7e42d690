// Attention over the 4-bit cache for sequences of many rows, codes as operands: f32, and what has no room for keys and values in T (kv_attention_prompts.hip).
//
// A workgroup has 16 MT rows for each of its waves, of one key head (new tokens times the query heads that share it), as columns of their
// matrix instructions, and goes through the tokens that they see 32 at a time. Codes are made operands once for all waves: a wave turns the codes of keys or of values of
// 16 tokens into numbers of 16 bits on their way into the LDS, in the order in which the instructions take them, scales and biases into f32; two stages, so that
// a block's codes come from memory while the one before is computed. Four tokens of one query to a lane (kv_attention.h), so that a scale is read
// once for MT of them. Bound by the vector units beside the matrix cores, a third of whose work is what goes into the LDS: four f32 prompts of 1000 tokens, 16 heads of 128
// values 122 us; a bf16 prompt of 8192 tokens, 32 heads, 942 us (583 TFLOP/s).
#include "kv_attention.h"

namespace mtq {

namespace {

template <int DT, int D, int G, int NW> struct TilesShape {
    static constexpr int Q = KvTerms<DT>::Q, NG = D / G, STEPS = D / 32, NT = G / 16, TH = 64 * NW;
    static constexpr int MT = D * Q <= 192 ? 2 : 1;   // sixteens of rows of a wave: sums and queries fill its registers
    static constexpr int ROWS = 16 * MT * NW;
    static constexpr int VT = 1024 + 16;                          // a tile of values, and what keeps the tiles' writes in different banks
    static constexpr int K = kBlock * D * 2, V = D / 16 * VT, S = 2 * NG * kBlock * 4;
    static constexpr int KSTAGE = K + S, VSTAGE = V + S;
    static constexpr int LDS = 2 * (KSTAGE + VSTAGE) + 8 * 4;
};

template <int DT, int D, int G, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void kv_tiles_kernel(KvAttentionArgs a, KvParts parts, uint32_t tiles) {
    using L = TilesShape<DT, D, G, NW>;
    using T = KvTerms<DT>;
    constexpr int MT = L::MT, NG = L::NG, NT = L::NT, STEPS = L::STEPS, TH = L::TH;
    constexpr int ITEMS = D / 2, RI = (ITEMS + 63) / 64, SI = (16 * NG + 63) / 64;   // pieces of 16 bytes of 16 tokens' codes, and a lane's of them and of the scales
    static_assert(NW == 4 || NW == 8, "");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const KvArgs& kv = a.kv;
    const uint32_t th = threadIdx.x, lane = th & 63u, wave = __builtin_amdgcn_readfirstlane(th >> 6), r = lane & 15u, g = lane >> 4;
    KvTile at_tile;
    if (!kv_tile<L::ROWS>(a, parts, tiles, at_tile)) return;
    const KvSeq& s = at_tile.s;
    const uint32_t shared = at_tile.shared, head = at_tile.head, rows = at_tile.rows, row0 = at_tile.row0, slice = at_tile.slice, slices = at_tile.slices;
    const uint32_t lo = at_tile.lo, hi = at_tile.hi, first_of_all = at_tile.first_end, b0 = at_tile.b0, b1 = at_tile.b1;
    auto end_of = [&](uint32_t i) { return kv_end(at_tile, i); };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    // This wave's rows, and a lane's.
    const uint32_t wave0 = row0 + wave * 16 * MT, wave_last = wave0 + 16 * MT - 1u < rows ? wave0 + 16 * MT - 1u : rows - 1u;
    const bool any = wave0 < rows;
    const uint32_t first_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave0) : 0u), last_end = __builtin_amdgcn_readfirstlane(any ? end_of(wave_last) : 0u);
    const uint32_t last_from = from_of(last_end);
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

    // A block's codes from memory into registers, and from there as operands into its stage. A wave brings the keys or the values of one of a block's two
    // sixteens of tokens, which lie on one page; of eight waves the first four have the even blocks.
    const uint32_t k16 = kv_sixteen<T::QK>(), v16 = kv_sixteen<DT_BF16>();
    const uint32_t half = wave & 1u, turn = wave / 4u;
    const bool values = wave & 2u;
    const uint8_t* const codes = (const uint8_t*)(values ? kv.v.codes : kv.k.codes);
    const void *const scales = values ? kv.v.scales : kv.k.scales, *const biases = values ? kv.v.biases : kv.k.biases;
    uint4 raw[RI];
    float sraw[SI], braw[SI];
    uint32_t raw_there = 0;   // whether what is in them is on a page
    // The pages of 64 of this wave's sixteens at a time, one to a lane: a scalar load would be waited for by whoever reads the LDS next.
    constexpr uint32_t STEP = NW / 4;
    uint32_t pages = 0, pages_from = 0;
    auto pages_at = [&](uint32_t b) {
        const uint32_t mine = b + lane * STEP, at = lo + mine * kBlock + 16 * half;
        pages_from = b;
        pages = mine < b1 && at < hi ? kv.pages[(uint64_t)s.seq * kv.pages_stride + (at >> kv.page_log2)] : 0xFFFFFFFFu;
    };
    auto fetch = [&](uint32_t b) {
        if ((b - pages_from) / STEP > 63u) pages_at(b);
        const uint32_t page = __builtin_amdgcn_readlane(pages, (b - pages_from) / STEP), at = lo + b * kBlock + 16 * half;
        raw_there = page < kv.n_pages;
        // (of no page: one that is there. The pool has fewer than 2^32 tokens and heads: host)
        const uint32_t slot = (((raw_there ? page : 0u) * kv.hkv + head) << kv.page_log2) + (at & ((1u << kv.page_log2) - 1u));
        const uint8_t* from_codes = codes + (uint64_t)slot * (D / 2);
#pragma unroll
        for (int u = 0; u < RI; u++) {
            const uint32_t i = u * 64 + lane;
            if (ITEMS % 64 == 0 || i < ITEMS) {
                if (values) {   // a word of each of four tokens
                    const uint32_t* p = (const uint32_t*)(from_codes + (i / (D / 8)) * (4 * (D / 2)) + i % (D / 8) * 4);
                    raw[u] = make_uint4(p[0], p[D / 8], p[2 * (D / 8)], p[3 * (D / 8)]);
                } else {        // four words of a token
                    raw[u] = *(const uint4*)(from_codes + i % 16 * (D / 2) + i / 16 * 16);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < SI; u++) {
            const uint32_t i = (u * 64 + lane) % (16 * NG);   // token and group
            sraw[u] = load_elem<DT>(scales, (uint64_t)slot * NG + i);
            braw[u] = load_elem<DT>(biases, (uint64_t)slot * NG + i);
        }
    };
    // [stage][sixteen]: bit 0: on a page (with the keys); bit 1: scales or biases that are no numbers (with the values)
    uint32_t* const flags = (uint32_t*)(lds + 2 * (L::KSTAGE + L::VSTAGE));
    auto store = [&](uint32_t b) {
        uint8_t* st = lds + (values ? 2 * L::KSTAGE + (b & 1u) * L::VSTAGE : (b & 1u) * L::KSTAGE);
#pragma unroll
        for (int u = 0; u < RI; u++) {
            const uint32_t i = u * 64 + lane, w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
            if (ITEMS % 64 == 0 || i < ITEMS) {
                if (values) {
                    const uint32_t quad = i / (D / 8), word = i % (D / 8);
                    uint8_t* to = st + (word / 2) * L::VT + (quad * 16 + word % 2 * 8) * 16 + half * 8;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        kr_u32x2 v;
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t two = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x0C000C00u | (uint32_t)(4 + e / 2) << 16 | (uint32_t)(e / 2));
                            v[j] = kv_operand<DT>(((e & 1 ? two >> 1 : two << 3) & 0x00780078u) | v16);
                        }
                        *(kr_u32x2*)(to + e * 16) = v;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        kr_u32x4 k;
#pragma unroll
                        for (int p = 0; p < 4; p++) k[p] = kv_operand<DT>(kv_pair<T::QK>(w[j], p, k16));
                        *(kr_u32x4*)(st + (half * STEPS * 64 + (i / 16) * 64 + j * 16 + i % 16) * 16) = k;   // (i / 16: step)
                    }
                }
            }
        }
        float* to = (float*)(st + (values ? L::V : L::K)) + 16 * half;   // [scales, biases - 16 scales of keys, + 8 scales of values][group][token]
        bool fine = true;
#pragma unroll
        for (int u = 0; u < SI; u++) {
            const uint32_t i = (u * 64 + lane) % (16 * NG);
            const bool in = raw_there && lo + b * kBlock + 16 * half + i / NG < hi;   // (where no token is: zeros)
            const float first = in ? sraw[u] : 0.f, second = in ? fmaf(values || T::CENTRED ? 8.f : -16.f, sraw[u], braw[u]) : 0.f;
            to[i % NG * kBlock + i / NG] = first;   // (by several lanes the same)
            to[(NG + i % NG) * kBlock + i / NG] = second;
            fine = fine && fabsf(first) < INFINITY && fabsf(second) < INFINITY;
        }
        const bool all_fine = __all(fine);
        if (lane == 0) flags[(values ? 4u : 0u) + (b & 1u) * 2u + half] = values ? !all_fine : raw_there;
    };

    kr_f32x4 o[MT][NG][NT] = {};
    float ones[MT][NG] = {}, bias[MT][NG] = {}, sum[MT] = {}, bar[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) bar[m] = -INFINITY;
    // A sixteen of a block's keys and their numbers, out of the LDS; and its scores.
    struct Keys {
        kr_u32x4 k[STEPS];
        kr_f32x4 s[NG], b[NG];
    };
    auto read_keys = [&](uint32_t b, int t, Keys& to) {
        const uint8_t* st = lds + (b & 1u) * L::KSTAGE;
        const float* sc = (const float*)(st + L::K) + 4 * g;
#pragma unroll
        for (int i = 0; i < STEPS; i++) to.k[i] = *(const kr_u32x4*)(st + (t * STEPS + i) * 1024 + lane * 16);
#pragma unroll
        for (int n = 0; n < NG; n++) {
            to.s[n] = *(const kr_f32x4*)(sc + n * kBlock + 16 * t);
            to.b[n] = *(const kr_f32x4*)(sc + (NG + n) * kBlock + 16 * t);
        }
    };
    auto scores = [&](const Keys& from, int t, float (&x)[MT][2][4]) {
#pragma unroll
        for (int n = 0; n < NG; n++) {
            kr_f32x4 acc[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) acc[m] = kr_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = n * (G / 32); i < (n + 1) * (G / 32); i++)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int e = T::Q - 1; e >= 0; e--) acc[m] = kr_mfma<T::QK>(from.k[i], q[m][e][i], acc[m]);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[m][t][i] = fmaf(from.b[n][i], qsum[m][n], n ? fmaf(from.s[n][i], acc[m][i], x[m][t][i]) : from.s[n][i] * acc[m][i]);
        }
    };
    // What a row does not see scores -inf; the bars are raised where scores pass them.
    uint32_t seen = 0xFFFFFFFFu;   // (8 bits for each m)
    bool whole = true, whole_of_all = true;   // (every row of the wave, and of the workgroup, sees all of the block)
    auto look = [&](uint32_t b, uint32_t there, float (&x)[MT][2][4]) {
        const uint32_t t0 = lo + b * kBlock;
        whole = t0 >= last_from && t0 + kBlock <= first_end && there == 3u;
        whole_of_all = t0 >= from_of(hi) && t0 + kBlock <= first_of_all && there == 3u;
        seen = 0xFFFFFFFFu;
        if (!whole) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t tok = t0 + 16 * t + 4 * g + i;
                        if (!((there >> t & 1u) && tok >= from[m] && tok < end[m])) {
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
    };
    // A weight of 0 does not keep a NaN out: where some rows of the workgroup do not see all of a block, values' scales and biases that are no numbers
    // become zeros, and the rows that see them have a NaN in that group's sum.
    auto take_out = [&](uint32_t b) {
        float* sc = (float*)(lds + 2 * L::KSTAGE + (b & 1u) * L::VSTAGE + L::V);
#pragma unroll
        for (int n = 0; n < NG; n++)
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float vs = sc[n * kBlock + 16 * t + 4 * g + i], vb = sc[(NG + n) * kBlock + 16 * t + 4 * g + i];
                    if (!(fabsf(vs) < INFINITY && fabsf(vb) < INFINITY)) {
#pragma unroll
                        for (int m = 0; m < MT; m++)
                            if (seen >> (8 * m + 4 * t + i) & 1u) bias[m][n] = __builtin_nanf("");
                    }
                }
        __syncthreads();
        for (uint32_t i = th; i < NG * kBlock; i += TH)
            if (!(fabsf(sc[i]) < INFINITY && fabsf(sc[NG * kBlock + i]) < INFINITY)) sc[i] = sc[NG * kBlock + i] = 0.f;
        __syncthreads();
    };
    // A block's weights out of its scores, one sixteen of them; a group's values and their numbers out of the LDS; p s as operands; and the values' sums.
    auto weigh = [&](int t, float (&x)[MT][2][4]) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float from_bar = bar[m] == -INFINITY ? 0.f : bar[m];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[m][t][i] = __builtin_amdgcn_exp2f(fmaf(x[m][t][i], c, -from_bar));
                sum[m] += x[m][t][i];
            }
        }
    };
    struct Values {
        kr_u32x4 v[NT];
        kr_f32x4 s[2], b[2];
    };
    auto read_values = [&](uint32_t b, int n, Values& to) {
        const uint8_t* st = lds + 2 * L::KSTAGE + (b & 1u) * L::VSTAGE;
        const float* sc = (const float*)(st + L::V) + 4 * g;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            to.s[t] = *(const kr_f32x4*)(sc + n * kBlock + 16 * t);
            to.b[t] = *(const kr_f32x4*)(sc + (NG + n) * kBlock + 16 * t);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) to.v[t] = *(const kr_u32x4*)(st + (n * NT + t) * L::VT + lane * 16);
    };
    auto operands = [&](const Values& from, int n, const float (&x)[MT][2][4], kr_u32x4 (&pt)[MT][T::P]) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) bias[m][n] = fmaf(x[m][t][i], from.b[t][i], bias[m][n]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float y[2][T::P];
#pragma unroll
                for (int e = 0; e < 2; e++) kv_split(x[m][j / 2][2 * j % 4 + e] * from.s[j / 2][2 * j % 4 + e], y[e]);
#pragma unroll
                for (int e = 0; e < T::P; e++) pt[m][e][j] = kv_pack_bf16(y[0][e], y[1][e]);
            }
        }
    };
    auto add_values = [&](const Values& from, int n, const kr_u32x4 (&pt)[MT][T::P]) {
        const kr_u32x4 less24 = {0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u};   // -24 in bf16
        kr_f32x4 less[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            less[m] = kr_f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (!T::CENTRED) {
#pragma unroll
                for (int e = T::P - 1; e >= 0; e--) less[m] = kr_mfma<DT_BF16>(less24, pt[m][e], less[m]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int e = T::P - 1; e >= 0; e--) o[m][n][t] = kr_mfma<DT_BF16>(from.v[t], pt[m][e], o[m][n][t]);
#pragma unroll
        for (int m = 0; m < MT; m++) ones[m][n] += less[m][0];
    };

    // The scores of a block are computed beside the values of the one before, so that the matrix cores have the one while the vector units have the
    // other. In turn b the keys of block b + 2 and the values of b + 1 go into the stages that turn b - 1 has read, and a wave's next codes are asked for.
    if (b0 < b1) {
        float x[MT][2][4];
        const uint32_t ahead = values ? 1u : 2u;
        uint32_t mine = b0 + (NW == 8 ? (b0 ^ turn) & 1u : 0u);   // this wave's next block
        pages_at(mine);
        fetch(mine);
        auto bring = [&](uint32_t upto) {   // this wave's blocks up to that one
            if (mine > upto || mine >= b1) return;
            store(mine);
            mine += STEP;
            if (mine < b1) fetch(mine);
        };
        bring(b0);
        if (!values) bring(b0 + 1u);
        __syncthreads();
        {
            Keys keys;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                read_keys(b0, t, keys);
                scores(keys, t, x);
            }
        }
        look(b0, __builtin_amdgcn_readfirstlane(flags[(b0 & 1u) * 2u] | flags[(b0 & 1u) * 2u + 1u] << 1), x);
        __syncthreads();
        for (uint32_t b = b0; b < b1; b++) {
            if (!whole_of_all) {
                const uint32_t* f = flags + 4u + (b & 1u) * 2u;
                if (__builtin_amdgcn_readfirstlane(f[0] | f[1])) take_out(b);
            }
            const uint32_t* f = flags + ((b + 1u) & 1u) * 2u;
            const uint32_t f0 = f[0], f1 = f[1];
            bring(b + ahead);
            // What the LDS is asked for in one part is used in the next (behind the last block the keys are those that are there, and not used).
            float next[MT][2][4];
            Keys first, second;
            Values group[2];
            kr_u32x4 pt[MT][T::P];
            read_keys(b + 1u, 0, first);
            weigh(0, x);
            __builtin_amdgcn_sched_barrier(0);
            read_keys(b + 1u, 1, second);
            scores(first, 0, next);
            weigh(1, x);
            __builtin_amdgcn_sched_barrier(0);
            read_values(b, 0, group[0]);
            scores(second, 1, next);
            __builtin_amdgcn_sched_barrier(0);
            operands(group[0], 0, x, pt);
#pragma unroll
            for (int n = 0; n < NG; n++) {
                if (n + 1 < NG) read_values(b, n + 1, group[(n + 1) & 1]);
                add_values(group[n & 1], n, pt);
                __builtin_amdgcn_sched_barrier(0);
                if (n + 1 < NG) operands(group[(n + 1) & 1], n + 1, x, pt);
            }
            if (b + 1u < b1) look(b + 1u, __builtin_amdgcn_readfirstlane(f0 | f1 << 1), next);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[m][t][i] = next[m][t][i];
            __syncthreads();
        }
    }

#pragma unroll
    for (int m = 0; m < MT; m++) {
        const float total = kv_column_sum(sum[m]);
        const uint32_t i = wave0 + 16 * m + r;
        const uint64_t at = (row_at[m] * a.hq + qh[m]) * parts.slices + slice;
        if (parts.slices > 1 && i < rows && g == 0) {
            if (slices > 1) {
                parts.sums[at * 2] = bar[m];
                parts.sums[at * 2 + 1] = total;
            }
            const uint32_t n = slices == 1 ? 0u : slices;   // (of one slice: nothing to join)
            if (slice + 1u == slices && n < parts.slices) parts.sums[(at - slice + n) * 2 + 1] = kNoMore;
        }
        const float by = slices > 1 ? 1.f : total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const float more = kv_column_sum(bias[m][n]) + ones[m][n];
            if (i >= rows) continue;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t d = n * G + 16 * t + 4 * g;
                kr_f32x4 v;
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = slices == 1 && total == 0.f ? 0.f : (o[m][n][t][j] + more) * by;
                if (slices > 1) {
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

// Waves of a workgroup: two to a SIMD, of heads of 256 values one, whose queries' terms and sums take all of its registers (six prompts of 3500 tokens, f32: 1800 us
// instead of 4130 with two that spill).
template <int D> constexpr int kWaves = D == 256 ? 4 : 8;

template <int DT, int D, int G> int launch(const KvAttentionArgs& p, KvParts parts, const LaunchCtx& lc) {
    using L = TilesShape<DT, D, G, kWaves<D>>;
    KvAttentionArgs a = p;
    static_assert(L::LDS <= 160 * 1024, "");
    const void* fn = (const void*)kv_tiles_kernel<DT, D, G, kWaves<D>>;
    const uint64_t tiles64 = kv_sets<L::ROWS>(a);
    if (tiles64 * a.kv.hkv * parts.slices > max_workgroups(64 * kWaves<D>)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    uint32_t tiles = (uint32_t)tiles64;
    LaunchCtx first = lc;
    if (parts.slices > 1) first.stop = nullptr;
    MTQ_HIP(set_max_dynamic_lds(fn, L::LDS));
    void* args[] = {&a, &parts, &tiles};
    MTQ_HIP(launch_kernel(fn, dim3(tiles * a.kv.hkv * parts.slices), dim3(64 * kWaves<D>), args, L::LDS, first));
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
    return 16 * (dim == 256 ? kWaves<256> : kWaves<128>) * (dim * (dtype == DT_F32 ? 3 : 1) <= 192 ? 2 : 1);
}

}  // namespace mtq
