// The gated delta rule token by token (gated_delta.h): single tokens, and sequences too short for chunks.
#include "gated_delta.h"

namespace mtq {

namespace {

// DKL: values of k a lane; WHOLE: dk = 16 DKL and every row on 16 bytes.
template <int DT, int DKL, bool WHOLE> __global__ __launch_bounds__(256) void delta_tokens_kernel(DeltaArgs a) {
    const uint32_t seq = blockIdx.x / a.hv, h = blockIdx.x % a.hv;
    const DeltaSeq s = delta_seq(a, seq);
    if (s.any) delta_tokens<DT, DKL, WHOLE>(a, s, h, (blockIdx.y * 4 + (threadIdx.x >> 6)) * 4);
}

template <int DT> const void* tokens_fn(uint32_t dk, bool whole) {
    if (whole && dk == 64) return (const void*)delta_tokens_kernel<DT, 4, true>;
    if (whole && dk == 128) return (const void*)delta_tokens_kernel<DT, 8, true>;
    if (whole && dk == 256) return (const void*)delta_tokens_kernel<DT, 16, true>;
    return dk <= 64 ? (const void*)delta_tokens_kernel<DT, 4, false> : dk <= 128 ? (const void*)delta_tokens_kernel<DT, 8, false>
                                                                                      : (const void*)delta_tokens_kernel<DT, 16, false>;
}

}  // namespace

int launch_delta_tokens(const DeltaArgs& p, const LaunchCtx& lc) {
    DeltaArgs a = p;
    const bool whole = delta_rows_whole(a);
    const void* fn = a.dtype == DT_F32 ? tokens_fn<DT_F32>(a.dk, whole) : a.dtype == DT_F16 ? tokens_fn<DT_F16>(a.dk, whole) : tokens_fn<DT_BF16>(a.dk, whole);
    void* args[] = {&a};
    MTQ_HIP(launch_kernel(fn, dim3(a.n_seqs * a.hv, (a.dv + 15) / 16), dim3(256), args, 0, lc));
    return ERR_OK;
}

}  // namespace mtq
