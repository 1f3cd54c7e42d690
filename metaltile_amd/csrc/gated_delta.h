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

}  // namespace mtq
