// Launches of the decode and join kernels of the packed cache's attention.
#include "mxq_capi_kv.h"

namespace {

template <int DT>
void launch(const KvAttnArgs& a, const mxq_kv::Plan& p, hipStream_t s) {
    // with a prompt kernel to follow, one more workgroup works out its stretches
    const unsigned grid = (unsigned)((p.whole ? p.decode_items : p.shares) * a.c.heads + (p.prompt ? 1 : 0));
    MXQ_KV_CASES(p.nb,
        constexpr int MOST = kv_decode_most_ct(NB, kv_terms<DT>());
        if (p.ct == 1) kv_decode_kernel<DT, NB, 1><<<grid, kThreads, 0, s>>>(a);
        else kv_decode_kernel<DT, NB, MOST><<<grid, kThreads, 0, s>>>(a))
}

template <int DT>
void launch_both_joins(const KvAttnArgs& a, const mxq_kv::Plan& p, hipStream_t s) {
    int64_t grid = a.join_blocks;
    MXQ_KV_CASES(p.nb,
        if (p.prompt && p.prompt_shares > 1) grid += p.prompt_items * a.c.heads * 4 * kv_prompt_ct(NB, kv_terms<DT>());
        KvAttnArgs part = a;
        for (int64_t first = 0; first < grid; first += mxq_kv::kMostWorkgroups) {
            const int64_t rest = grid - first;
            part.join_first = (int)first;
            kv_join_kernel<DT, NB><<<(unsigned)(rest < mxq_kv::kMostWorkgroups ? rest : mxq_kv::kMostWorkgroups), kThreads, 0, s>>>(part);
        })
}

}  // namespace

namespace mxq_kv {
void launch_decode(int dtype, const void* args, const Plan& p, hipStream_t s) {      // (KvAttnArgs has no linkage)
    const KvAttnArgs& a = *reinterpret_cast<const KvAttnArgs*>(args);
    if (dtype == MXQ_DTYPE_BF16) launch<MXQ_BF16>(a, p, s);
    else launch<MXQ_F16>(a, p, s);
}
void launch_join(int dtype, const void* args, const Plan& p, hipStream_t s) {
    const KvAttnArgs& a = *reinterpret_cast<const KvAttnArgs*>(args);
    if (dtype == MXQ_DTYPE_BF16) launch_both_joins<MXQ_BF16>(a, p, s);
    else launch_both_joins<MXQ_F16>(a, p, s);
}
}  // namespace mxq_kv
