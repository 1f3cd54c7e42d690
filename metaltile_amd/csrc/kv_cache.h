// A paged cache of keys and values in packed 4-bit codes, as its writer, reader and attention see it.
//
// A page holds page_size tokens of every key head. Codes, scales and biases are the packed format's (mtq_affine_quantize, 4 bits): of a token's
// head_dim values of a head, eight codes a word from its lowest bits on, and a scale and a bias in T for each group along the head;
// value = scale * code + bias. Keys and values have three arrays each:
//   codes u32 [n_pages, heads, page_size, dim / 8], scales / biases T [n_pages, heads, page_size, dim / group]
// Token p of sequence i lies on page pages[i][p / page_size]; an id >= n_pages names no page. Sequence i has lens[i] tokens, the
// new ones (offsets[i] .. offsets[i + 1] - 1 of the call's rows) among them, which are its last.
#pragma once
#include "mtq_device.h"
#include "mtq_internal.h"

namespace mtq {

// The number of entries of a[0 .. n) (ascending) that are not above t: a wave asks 64 places at a time. The same in every lane; all lanes call.
__device__ __forceinline__ uint32_t kv_count_upto(const uint32_t* a, uint32_t n, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0;
    while (n) {
        const uint32_t step = (n + 63u) / 64u;   // a lane asks for the last entry of its piece of `step`
        const uint32_t at = (lane + 1u) * step - 1u;
        const bool in = at < n && a[lo + at] <= t;
        const uint32_t whole = (uint32_t)__popcll(__ballot(in));   // pieces that are not above t from end to end
        lo += whole * step;
        n = whole * step < n ? (step == 1 ? 0u : (n - whole * step < step ? n - whole * step : step)) : 0u;
    }
    return lo;
}

struct KvSeq {
    uint32_t seq, first_row, rows, len;   // its new tokens are rows first_row .. first_row + rows - 1 of the call; tokens in all
};
// Sequence i (below n_seqs).
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, uint32_t i) {
    KvSeq s;
    s.seq = i;
    if (a.offsets) {
        const uint32_t lo = a.offsets[i], hi = a.offsets[i + 1];
        s.first_row = lo < a.n_tokens ? lo : a.n_tokens;
        const uint32_t end = hi < a.n_tokens ? hi : a.n_tokens;
        s.rows = end > s.first_row ? end - s.first_row : 0u;
    } else {
        s.rows = a.n_tokens / a.n_seqs;
        s.first_row = i * s.rows;
    }
    const uint32_t len = a.lens[i];
    s.len = len < a.max_len ? len : a.max_len;
    return s;
}

}  // namespace mtq
