// Launch of the prompt kernel of the packed cache's attention.
#include "mxq_capi_kv.h"

namespace {

template <int DT>
void launch(const KvAttnArgs& a, const mxq_kv::Plan& p, hipStream_t s) {
    const unsigned grid = (unsigned)(p.prompt_shares * a.c.heads);
    MXQ_KV_CASES(p.nb,
        constexpr int CT = kv_prompt_ct(NB, kv_terms<DT>());
        if (a.out_wide) kv_prompt_kernel<DT, NB, CT, true><<<grid, kThreads, 0, s>>>(a);
        else kv_prompt_kernel<DT, NB, CT, false><<<grid, kThreads, 0, s>>>(a))
}

}  // namespace

namespace mxq_kv {
void launch_prompt(int dtype, const void* args, const Plan& p, hipStream_t s) {      // (KvAttnArgs has no linkage)
    const KvAttnArgs& a = *reinterpret_cast<const KvAttnArgs*>(args);
    if (dtype == MXQ_DTYPE_BF16) launch<MXQ_BF16>(a, p, s);
    else launch<MXQ_F16>(a, p, s);
}
}  // namespace mxq_kv
