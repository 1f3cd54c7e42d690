// Which kernel a call of the attention over the 4-bit cache takes, and into how many slices its tokens are cut.
#include "kv_attention.h"

namespace mtq {

static uint32_t num_cus() {
    static int n = 0;
    if (n == 0) {
        int dev = 0, v = 0;
        n = (hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) ? v : 256;
    }
    return (uint32_t)n;
}

KvPlan kv_attention_plan(int dtype, const KvAttentionArgs& a) {
    KvPlan p;
    const uint64_t units = (uint64_t)a.kv.n_seqs * a.kv.hkv, cus = num_cus();
    const uint32_t span = a.window && a.window < a.kv.max_len ? a.window : a.kv.max_len;   // tokens that a row sees at most
    p.large = units < 2 * cus;
    const uint64_t want = ((p.large ? 1 : 4) * cus + units - 1) / units, most = span / (p.large ? 1024 : 512);
    p.slices = (uint32_t)(want < most ? want : most);
    if (options().kv_waves) p.large = options().kv_waves == 2;
    if (options().kv_slices) p.slices = (uint32_t)options().kv_slices;
    if (p.slices < 1) p.slices = 1;
    while (p.slices > 1 && units * p.slices > max_workgroups(1024)) p.slices--;
    p.scratch = p.slices > 1 ? (size_t)a.kv.n_tokens * a.hq * p.slices * (a.kv.dim + 2) * sizeof(float) : 0;
    return p;
}

int launch_kv_attention(int dtype, const KvAttentionArgs& a, const KvPlan& plan, void* scratch, const LaunchCtx& lc) {
    KvParts parts;
    parts.slices = scratch ? plan.slices : 1;
    parts.values = (float*)scratch;
    parts.sums = scratch ? parts.values + (size_t)a.kv.n_tokens * a.hq * parts.slices * a.kv.dim : nullptr;
    if ((uint64_t)a.kv.n_seqs * a.kv.hkv * parts.slices > max_workgroups(1024)) return fail(ERR_SHAPE, "more sequences and heads than a launch can have workgroups");
    return launch_kv_rows(dtype, a, parts, plan.large, lc);
}

}  // namespace mtq
