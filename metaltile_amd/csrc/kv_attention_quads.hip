// Attention over the 4-bit cache for up to four rows a sequence and key head (a decode step): bound by the cache's way from memory.
//
// With four rows the columns of a 16-row instruction would be empty for the most part, and so would the lanes' work on scores and scales, which is
// what the vector units have most of: 419 instructions for 32 tokens (kv_attention_rows.hip), here 684 for 64. The instruction is the one of sixteen 4 x 4 x 4 products, and a
// lane has a token: 64 of them at a time, each lane with its own scale and bias, and the scores of four queries.
//   scores  block b has tokens 4 b .. 4 b + 3 as columns, and four queries as rows, the same for all blocks: their numbers lie in the lanes once, four to a
//           block, and the instruction takes block j's for all (its broadcast of A)
//   values  rows are queries again, the sum goes over four tokens of a block, and its columns are numbers of four words: in sixteen lanes the words of
//           128 numbers, for the sixteen tokens that these lanes have weights of. p s of four tokens is turned from lane = token to lane = query inside a block; which
//           tokens a block multiplies goes round with k, so that each block of a group's words has p times that group's scale
// Tokens lie in the LDS by rows. Of values those of a quad are in an order turned by their sixteen, of keys a row's pieces of 16 bytes in one turned by its place, which keeps
// reads of both free of bank conflicts. A block's keys are asked for again as soon as they are in registers, and so are its values.
// 64 sequences of 4096 tokens, 8 heads of 128 values, bf16: 63 us uncut (4.8 TB/s; 16 rows to a wave: 74), 256 of them 220 us (5.5 TB/s); of 1 to 8192 tokens 72 us, of which
// the join is 5; one of 131071 tokens, f16: 40 us (3.6 TB/s).
#include "kv_attention.h"

namespace mtq {

namespace {

typedef short kq_s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 kq_f16x4 __attribute__((ext_vector_type(4)));

template <int QK, int CBSZ, int ABID> __device__ __forceinline__ kr_f32x4 kq_mfma(kr_u32x2 a, kr_u32x2 b, kr_f32x4 c) {
    if constexpr (QK == DT_BF16) return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(__builtin_bit_cast(kq_s16x4, a), __builtin_bit_cast(kq_s16x4, b), c, CBSZ, ABID, 0);
    else return __builtin_amdgcn_mfma_f32_4x4x4f16(__builtin_bit_cast(kq_f16x4, a), __builtin_bit_cast(kq_f16x4, b), c, CBSZ, ABID, 0);
}

template <int DT, int D, int G> struct QuadsLds {
    static constexpr int ES = DT == DT_F32 ? 4 : 2, NG = D / G, ROWS = 4;
    static constexpr int CODES = 32 * D;                                // of 64 tokens' keys, or values
    static constexpr int SIXTEEN = 16 * NG * ES;                        // scales, or biases, of 16 tokens
    static constexpr int LOADS = SIXTEEN * 4 > 256 ? SIXTEEN * 4 / 256 : 1;   // that bring 64 tokens' scales, or biases
    static constexpr int PART = CODES + 2 * LOADS * 256;
    static constexpr int JOIN = ROWS * (D + 4) * 4;
    static constexpr int WAVE = 2 * PART > JOIN ? 2 * PART : JOIN;
    // Waves of a SIMD, by the registers: with more of them an instance spills (f32, 256 values in groups of 32: 295 us with one, 663 with two).
    static constexpr int AT_ONCE = D == 256 && (G == 32 || (DT == DT_F32 && G == 64)) ? 1 : DT == DT_F32 || D > 128 ? 2 : 3;
    static_assert(4 * WAVE <= 160 * 1024, "");
};

template <int DT, int D, int G>
__global__ __launch_bounds__(256, (QuadsLds<DT, D, G>::AT_ONCE)) void kv_quads_kernel(KvAttentionArgs a, KvParts parts) {
    using L = QuadsLds<DT, D, G>;
    using T = KvTerms<DT>;
    constexpr int QS = 1, NW = 4, NG = L::NG, ES = L::ES, WORDS = D / 8, ROWS = L::ROWS;
    constexpr int PASSES = D == 256 ? 2 : 1;             // of 128 numbers' words over sixteen lanes
    constexpr int GROUPS = NG / PASSES;                  // of a pass
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const KvArgs& kv = a.kv;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block4 = lane / 4u % 4u, sixteen = lane / 16u;
    const uint32_t head = blockIdx.x % kv.hkv, shared = a.hq / kv.hkv;
    KvPiece piece;
    if (!kv_piece<L::ROWS>(a, parts, blockIdx.x / kv.hkv, piece)) return;   // (all of the workgroup's waves find the same)
    const KvSeq& s = piece.s;
    const uint32_t slice = piece.slice, slices = piece.slices;
    uint8_t* mine = lds + wave * L::WAVE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
    const uint32_t rows = s.rows * shared;
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);   // (not 0: what is hidden scores -inf)
    const uint32_t k16 = kv_sixteen<T::QK>(), v16 = kv_sixteen<DT_BF16>();
    // p s, turned within a block of four lanes: which halves and which order.
    const uint32_t turn = lane & 1u ? 0x03020706u : 0x05040100u;

    const uint32_t row0 = piece.set * ROWS;
    const uint32_t count = rows - row0 < (uint32_t)ROWS ? rows - row0 : (uint32_t)ROWS;
    auto end_of = [&](uint32_t i) { const int32_t e = (int32_t)(s.len + i / shared + 1u) - (int32_t)s.rows; return e > 0 ? (uint32_t)e : 0u; };
    auto from_of = [&](uint32_t e) { return a.window && e > a.window ? e - a.window : 0u; };
    uint32_t end[ROWS];   // a row sees tokens from_of(end) .. end - 1
#pragma unroll
    for (int i = 0; i < ROWS; i++) end[i] = __builtin_amdgcn_readfirstlane(end_of(row0 + (i < (int)count ? i : count - 1u)));
    const uint32_t first_end = end[0], last_end = end[ROWS - 1], lo = from_of(first_end) & ~15u, last_from = from_of(last_end);
    const uint32_t blocks = kv.n_pages && last_end > lo ? (last_end - lo + 63u) / 64u : 0u;
    const uint32_t workers = slices * NW, per = (blocks + workers - 1u) / workers;
    const uint32_t b0 = (slice * NW + wave) * per < blocks ? (slice * NW + wave) * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;

    // Pages of 64 sixteens of tokens at a time, one to a lane.
    uint32_t page = 0, page_from = 0;
    auto pages_at = [&](uint32_t h) {
        page_from = h;
        const uint32_t at = (h + lane) * 16u;
        page = at < last_end ? kv.pages[(uint64_t)s.seq * kv.pages_stride + (at >> kv.page_log2)] : 0xFFFFFFFFu;
    };
    // A part of a block (keys or values: codes, scales, biases) into the LDS.
    auto issue = [&](uint32_t b, int part) {
        const uint32_t h = lo / 16u + 4u * b;
        uint32_t slot[4];   // [page, head, place] (of no page: one that is there; a pool has fewer than 2^32: host)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pg = __builtin_amdgcn_readlane(page, h + i - page_from), p = pg < kv.n_pages ? pg : 0u;
            slot[i] = ((p * kv.hkv + head) << kv.page_log2) + (((h + i) * 16u) & ((1u << kv.page_log2) - 1u));
        }
        const uint8_t* codes = (const uint8_t*)(part ? kv.v.codes : kv.k.codes);
        const uint8_t *scales = (const uint8_t*)(part ? kv.v.scales : kv.k.scales), *biases = (const uint8_t*)(part ? kv.v.biases : kv.k.biases);
        const uint32_t to = lds0 + part * L::PART;
        constexpr uint32_t PIECES = D / 32;   // of 16 bytes of a token
#pragma unroll
        for (int u = 0; u < D / 32; u++) {    // 64 pieces in turn: by token (those of a quad turned by their sixteen), then piece
            const uint32_t p = u * 64 + lane, row = p / PIECES, x = row / 16, piece = part ? p % PIECES : p % PIECES ^ (row * PIECES / 16) % PIECES;
            const uint32_t at = slot[u * 64 / (16 * PIECES)];
            kv_load16(__builtin_amdgcn_readfirstlane(to + u * 1024), codes + (uint64_t)(at + (row % 16 ^ x)) * (D / 2) + piece * 16);
        }
#pragma unroll
        for (int array = 0; array < 2; array++)
#pragma unroll
            for (int u = 0; u < L::LOADS; u++) {
                const uint32_t p = (u * 256 + lane * 4) % (L::SIXTEEN * 4), x = p / L::SIXTEEN;
                const uint32_t at = x & 2u ? (x & 1u ? slot[3] : slot[2]) : (x & 1u ? slot[1] : slot[0]);
                kv_load4(__builtin_amdgcn_readfirstlane(to + L::CODES + (array * L::LOADS + u) * 256), (array ? biases : scales) + (uint64_t)at * (NG * ES) + p % L::SIXTEEN);
            }
    };
    // The first keys and values are on their way while the queries come.
    auto room = [&](uint32_t b) {   // the pages of block b's four sixteens
        const uint32_t h = lo / 16u + 4u * b;
        if (h + 3u - page_from > 63u) pages_at(h);
    };
    if (b0 < b1) {
        pages_at(lo / 16u + 4u * b0);
        issue(b0, 0);
        issue(b0, 1);
    }

    // Queries: row i of a block; block j of sixteen has a half of word j / 2's numbers, in the order in which a word's nibbles come out.
    kr_u32x2 q[QS][T::Q][D / 64];
    float qsum[ROWS][NG];
#pragma unroll
    for (int m = 0; m < QS; m++) {
        uint32_t i = row0 + 4 * m + (lane & 3u);
        if (i >= rows) i = rows - 1u;
        const uint64_t at = (uint64_t)(s.first_row + i / shared) * a.q_stride + (uint64_t)(head * shared + i % shared) * D + lane / 8 * 8 + (lane & 4u ? 2 : 0);
        float part[NG] = {};
#pragma unroll
        for (int j = 0; j < D / 64; j++) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = load_elem<DT>(a.q, at + 64 * j + (e & 1) * 4 + e / 2);
                if (a.scale < 0.f) v[e] = -v[e];
            }
            if constexpr (DT == DT_F16) {
                q[m][0][j] = kr_u32x2{(uint32_t)f32_to_elem_bits<DT_F16>(v[0]) | (uint32_t)f32_to_elem_bits<DT_F16>(v[1]) << 16,
                                      (uint32_t)f32_to_elem_bits<DT_F16>(v[2]) | (uint32_t)f32_to_elem_bits<DT_F16>(v[3]) << 16};
            } else {
                float t[4][T::Q];
#pragma unroll
                for (int e = 0; e < 4; e++) kv_split(v[e], t[e]);
#pragma unroll
                for (int e = 0; e < T::Q; e++) q[m][e][j] = kr_u32x2{kv_pack_bf16(t[0][e], t[1][e]), kv_pack_bf16(t[2][e], t[3][e])};
            }
            const float four = (v[0] + v[1]) + (v[2] + v[3]);
            if constexpr (G == 32) {   // (lanes 0..31 have the lower 32 of these 64 numbers)
                part[2 * j] += lane < 32 ? four : 0.f;
                part[2 * j + 1] += lane < 32 ? 0.f : four;
            } else {
                part[64 * j / G] += four;
            }
        }
        // Sums over the lanes of a row (lane & 3), and then the four rows' as numbers that all lanes have.
#pragma unroll
        for (int n = 0; n < NG; n++) {
            float v = part[n];
            v += __shfl_xor(v, 4, 64);
            v += __shfl_xor(v, 8, 64);
            v = kv_column_sum(v);
#pragma unroll
            for (int r = 0; r < 4; r++) qsum[4 * m + r][n] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), r));
        }
    }

    kr_f32x4 o[QS][PASSES][8] = {}, ones[QS][PASSES] = {};   // values of a lane's word, rows r; -24 sum p s of its group
    float bias[ROWS][NG] = {}, sum[ROWS] = {}, bar[ROWS];       // (a lane's tokens')
#pragma unroll
    for (int i = 0; i < ROWS; i++) bar[i] = -INFINITY;

    constexpr int ON_WAY = D / 32 + 2 * L::LOADS;   // loads of a part
    // This lane's token's numbers of a part.
    struct Numbers {
        uint32_t w[NG * ES >= 4 ? NG * ES / 4 : 1];
        __device__ __forceinline__ float operator()(int n) const {
            if constexpr (DT == DT_F32) return __uint_as_float(w[n]);
            else return kr_elem<DT>(w[n / 2], n & 1);
        }
    };
    auto numbers = [&](const uint8_t* p) {
        Numbers v;
        if constexpr (NG * ES == 2) {
            v.w[0] = *(const uint16_t*)(p + lane * 2);
        } else {
#pragma unroll
            for (int i = 0; i < NG * ES / 4; i++) v.w[i] = *(const uint32_t*)(p + lane * (NG * ES) + 4 * i);
        }
        return v;
    };
    for (uint32_t b = b0; b < b1; b++) {
        // ---- scores
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ON_WAY) : "memory");   // (the values' loads are behind the keys')
        const uint32_t t0 = lo + 64u * b, h = lo / 16u + 4u * b;
        const uint32_t my_page = (uint32_t)__shfl((int)page, (int)(h - page_from + sixteen), 64);
        uint4 kw[WORDS / 4];
        const uint8_t* row = mine + (lane ^ sixteen) * (D / 2);
        const uint32_t turned = (lane ^ sixteen) * (D / 32) / 16 % (D / 32);
#pragma unroll
        for (int i = 0; i < WORDS / 4; i++) kw[i] = *(const uint4*)(row + 16 * (i ^ turned));
        const Numbers ks = numbers(mine + L::CODES), kb = numbers(mine + L::CODES + L::LOADS * 256);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (b + 1u < b1) {
            room(b + 1u);
            issue(b + 1u, 0);
        }
        float x[ROWS];
        kr_for<0, NG>([&](auto group) {   // (an instruction names its block by a constant)
            constexpr int n = decltype(group)::value;
            kr_f32x4 acc[QS] = {};
            auto step = [&](auto word) {
                constexpr int W = decltype(word)::value;
                const uint4& four = kw[W / 4];
                const uint32_t w = W % 4 == 0 ? four.x : W % 4 == 1 ? four.y : W % 4 == 2 ? four.z : four.w;
                auto pair = [&](int p) { return kv_operand<DT>(kv_pair<T::QK>(w, p, k16)); };
                const kr_u32x2 first = {pair(0), pair(1)}, second = {pair(2), pair(3)};
#pragma unroll
                for (int m = 0; m < QS; m++)
#pragma unroll
                    for (int e = T::Q - 1; e >= 0; e--) {
                        acc[m] = kq_mfma<T::QK, 4, W % 8 * 2>(q[m][e][W / 8], first, acc[m]);
                        acc[m] = kq_mfma<T::QK, 4, W % 8 * 2 + 1>(q[m][e][W / 8], second, acc[m]);
                    }
            };
            kr_for<n * G / 8, (n + 1) * G / 8>(step);
            const float sc = ks(n), rest = fmaf(T::CENTRED ? 8.f : -16.f, sc, kb(n));
#pragma unroll
            for (int i = 0; i < ROWS; i++) x[i] = fmaf(rest, qsum[i][n], n ? fmaf(sc, acc[i / 4][i % 4], x[i]) : sc * acc[i / 4][i % 4]);
        });
        const bool whole = t0 >= last_from && t0 + 64u <= first_end && __all(my_page < kv.n_pages);
        uint32_t seen = 0xFFu;   // (a bit for each row)
        if (!whole) {
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                if (!(my_page < kv.n_pages && t0 + lane >= from_of(end[i]) && t0 + lane < end[i])) {
                    x[i] = -INFINITY;
                    seen &= ~(1u << i);
                }
        }
        bool over = false;
#pragma unroll
        for (int i = 0; i < ROWS; i++) over = over || x[i] * c > bar[i] + kSlack;
        if (__any(over)) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                float top = x[i];
                top = fmaxf(top, dpp_f32<0xB1>(top));
                top = fmaxf(top, dpp_f32<0x4E>(top));
                top = fmaxf(top, dpp_f32<0x141>(top));
                top = kv_column_max(fmaxf(top, dpp_f32<0x140>(top)));
                const float to = fmaxf(bar[i], top * c), keep = to > bar[i] ? __builtin_amdgcn_exp2f(bar[i] - to) : 1.f;
                sum[i] *= keep;
#pragma unroll
                for (int n = 0; n < NG; n++) bias[i][n] *= keep;
#pragma unroll
                for (int p = 0; p < PASSES; p++) {
                    ones[i / 4][p][i % 4] *= keep;
#pragma unroll
                    for (int e = 0; e < 8; e++) o[i / 4][p][e][i % 4] *= keep;
                }
                bar[i] = to;
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, bar[i] == -INFINITY ? 0.f : -bar[i]));
            sum[i] += x[i];
        }
        // ---- values
        if (b + 1u < b1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ON_WAY) : "memory");   // (the next keys' loads are behind these)
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t* vt = mine + L::PART;
        Numbers vs = numbers(vt + L::CODES), vb = numbers(vt + L::CODES + L::LOADS * 256);
        uint32_t w[PASSES][4][4];   // [pass][k][token of the quad]: a lane's word of tokens 16 sixteen + 4 ((block - k) & 3) + t
#pragma unroll
        for (int p = 0; p < PASSES; p++)
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    w[p][k][t] = *(const uint32_t*)(vt + (16 * sixteen + 4 * ((block4 - k) & 3u) + (t ^ sixteen)) * (D / 2) + (p * 16 + lane % 16) * 4);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (b + 1u < b1) issue(b + 1u, 1);
        float ps[ROWS][NG];
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const float sc = vs(n);
            float more = fmaf(8.f, sc, vb(n));
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                ps[i][n] = x[i] * sc;
                if (whole) {
                    bias[i][n] = fmaf(x[i], more, bias[i][n]);
                } else {   // (a weight of 0 does not keep a NaN out)
                    const bool yes = seen >> i & 1u;
                    ps[i][n] = yes ? ps[i][n] : 0.f;
                    bias[i][n] = yes ? fmaf(x[i], more, bias[i][n]) : bias[i][n];
                }
            }
        }
#pragma unroll
        for (int m = 0; m < QS; m++)
#pragma unroll
            for (int p = 0; p < PASSES; p++) {
                // [k][term]: what this lane's block multiplies in turn k
                kr_u32x2 at[4][T::P];
                kr_for<0, GROUPS>([&](auto group) {
                    constexpr int n = decltype(group)::value;
                    constexpr int MASK = (0 == n ? 1 : 0) | (GROUPS / 4 == n ? 2 : 0) | (2 * GROUPS / 4 == n ? 4 : 0) | (3 * GROUPS / 4 == n ? 8 : 0);   // blocks of this group's words
                    float t[4][T::P];
#pragma unroll
                    for (int r = 0; r < 4; r++) kv_split(ps[4 * m + r][p * GROUPS + n], t[r]);
#pragma unroll
                    for (int e = 0; e < T::P; e++) {
                        // From four rows of a token to four tokens of a row, inside four lanes: rows 0, 1 | 2, 3 against the lanes two apart, then neighbours.
                        const uint32_t u0 = kv_pack_bf16(t[0][e], t[1][e]), u1 = kv_pack_bf16(t[2][e], t[3][e]);
                        const bool upper = lane & 2u;
                        const uint32_t keep = upper ? u1 : u0, send = upper ? u0 : u1;
                        const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0x4E, 0xF, 0xF, true);
                        const uint32_t keep_by = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)keep, 0xB1, 0xF, 0xF, true);
                        const uint32_t got_by = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)got, 0xB1, 0xF, 0xF, true);
                        const uint32_t own = __builtin_amdgcn_perm(keep_by, keep, turn), other = __builtin_amdgcn_perm(got_by, got, turn);
                        const uint32_t z[2] = {upper ? other : own, upper ? own : other};
                        // In turn k a block has the tokens of the block k before (of the four it goes round).
                        kr_for<0, 4>([&](auto turns) {
                            constexpr int k = decltype(turns)::value, ctrl = k ? 0x120 + 4 * k : 0xE4;
#pragma unroll
                            for (int d = 0; d < 2; d++)
                                at[k][e][d] = (uint32_t)__builtin_amdgcn_update_dpp(n ? (int)at[k][e][d] : (int)z[d], (int)z[d], ctrl, 0xF, MASK, false);
                        });
                    }
                });
                const kr_u32x2 less24 = {0xC1C0C1C0u, 0xC1C0C1C0u};   // -24 in bf16
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (!T::CENTRED) {
#pragma unroll
                        for (int e = T::P - 1; e >= 0; e--) ones[m][p] = kq_mfma<DT_BF16, 0, 0>(at[k][e], less24, ones[m][p]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const uint32_t sel = 0x0C000C00u | (uint32_t)(4 + i / 2) << 16 | (uint32_t)(i / 2);
                        const uint32_t y0 = __builtin_amdgcn_perm(w[p][k][1], w[p][k][0], sel), y1 = __builtin_amdgcn_perm(w[p][k][3], w[p][k][2], sel);
                        auto pair = [&](uint32_t y) { return kv_operand<DT>((y & 0x00780078u) | v16); };
                        const kr_u32x2 even = {pair(y0 << 3), pair(y1 << 3)}, odd = {pair(y0 >> 1), pair(y1 >> 1)};
#pragma unroll
                        for (int e = T::P - 1; e >= 0; e--) {
                            o[m][p][i] = kq_mfma<DT_BF16, 0, 0>(at[k][e], even, o[m][p][i]);
                            o[m][p][i + 1] = kq_mfma<DT_BF16, 0, 0>(at[k][e], odd, o[m][p][i + 1]);
                        }
                    }
                }
            }
    }

    // The lanes' sums into the LDS, relative to the wave's bars; the waves' joined.
    float* join = (float*)mine;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float total = seg_allreduce(sum[i], 64);
        float more[NG];
#pragma unroll
        for (int n = 0; n < NG; n++) more[n] = seg_allreduce(bias[i][n], 64);
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const float less = kv_column_sum(ones[i / 4][p][i % 4]);
            float mine_more = more[p * GROUPS];
#pragma unroll
            for (int n = 1; n < GROUPS; n++) mine_more = block4 * GROUPS / 4 == (uint32_t)n ? more[p * GROUPS + n] : mine_more;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = kv_column_sum(o[i / 4][p][e][i % 4]) + less + mine_more;
                if (sixteen == 0) join[i * (D + 4) + (p * 16 + lane % 16) * 8 + e] = v;
            }
        }
        if (lane == 0) {
            join[i * (D + 4) + D] = bar[i];
            join[i * (D + 4) + D + 1] = total;
        }
    }
    __syncthreads();
    for (uint32_t u = threadIdx.x; u < count * (D / 4); u += 64 * NW) {
        const uint32_t r = u / (D / 4), d = u % (D / 4) * 4, i = row0 + r, tok = s.first_row + i / shared, h = head * shared + i % shared;
        const float* all = (const float*)lds + r * (D + 4);
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, all[w * (L::WAVE / 4) + D]);
        kr_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float* one = all + w * (L::WAVE / 4);
            const float part = one[D + 1], f = one[D] == -INFINITY ? (part == 0.f ? 0.f : 1.f) : exp2f(one[D] - top);   // (no bar and a sum: NaN)
            total = fmaf(part, f, total);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = f == 0.f && part == 0.f ? v[j] : fmaf(one[d + j], f, v[j]);
        }
        if (slices == 1) {
            const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int j = 0; j < 4; j++) store_elem<DT>(a.out, (uint64_t)tok * a.out_stride + (uint64_t)h * D + d + j, total == 0.f ? 0.f : v[j] * inv);
        } else {
            const uint64_t at = ((uint64_t)tok * a.hq + h) * parts.slices + slice;
            *(kr_f32x4*)(parts.values + at * D + d) = v;
            if (d == 0) {
                parts.sums[at * 2] = top;
                parts.sums[at * 2 + 1] = total;
            }
        }
        if (d == 0 && slice + 1u == slices && parts.slices > 1) {   // (of one slice: nothing to join)
            const uint32_t n = slices == 1 ? 0u : slices;
            if (n < parts.slices) parts.sums[(((uint64_t)tok * a.hq + h) * parts.slices + n) * 2 + 1] = kNoMore;
        }
    }
}

template <int DT, int D, int G> int launch(const KvAttentionArgs& p, KvParts parts, const LaunchCtx& lc) {
    KvAttentionArgs a = p;
    const void* fn = (const void*)kv_quads_kernel<DT, D, G>;
    const size_t bytes = 4 * QuadsLds<DT, D, G>::WAVE;
    const uint64_t groups = kv_pieces<4>(a, parts);
    if (groups * a.kv.hkv > max_workgroups(256)) return fail(ERR_SHAPE, "more rows and heads than a launch can have workgroups");
    LaunchCtx first = lc, last = lc;
    if (parts.slices > 1) {
        first.stop = nullptr;
        last.start = nullptr;
    }
    MTQ_HIP(set_max_dynamic_lds(fn, bytes));
    void* args[] = {&a, &parts};
    MTQ_HIP(launch_kernel(fn, dim3((uint32_t)(groups * a.kv.hkv)), dim3(256), args, bytes, first));
    return parts.slices > 1 ? launch_kv_join(DT, a, parts, last) : ERR_OK;
}

template <int DT> int launch_of(const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (p.kv.dim * 1000 + p.kv.group) {
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

int launch_kv_quads(int dtype, const KvAttentionArgs& p, const KvParts& parts, const LaunchCtx& lc) {
    switch (dtype) {
        case DT_F32: return launch_of<DT_F32>(p, parts, lc);
        case DT_F16: return launch_of<DT_F16>(p, parts, lc);
        default: return launch_of<DT_BF16>(p, parts, lc);
    }
}

}  // namespace mtq
