// Launches of the decode and join kernels of the packed cache's attention.
#include "mxq_capi_kv.h"

namespace {

template <int DT>
void launch(const KvAttnArgs& a, const mxq_kv::Plan& p, hipStream_t s) {
    const unsigned grid = (unsigned)((p.whole ? p.decode_items : p.shares) * a.c.heads);
    MXQ_KV_CASES(p.nb,
        if (p.ct == 1) kv_decode_kernel<DT, NB, 1><<<grid, kThreads, 0, s>>>(a);
        else kv_decode_kernel<DT, NB, 2><<<grid, kThreads, 0, s>>>(a))
    if (p.whole) return;
    const unsigned rows = (unsigned)(a.rows * a.c.heads * a.group);
    MXQ_KV_CASES(p.nb, kv_join_kernel<DT, NB><<<rows, kThreads, 0, s>>>(a))
}

}  // namespace

namespace mxq_kv {
void launch_decode(int dtype, const void* args, const Plan& p, hipStream_t s) {      // (KvAttnArgs has no linkage)
    const KvAttnArgs& a = *reinterpret_cast<const KvAttnArgs*>(args);
    if (dtype == MXQ_DTYPE_BF16) launch<MXQ_BF16>(a, p, s);
    else launch<MXQ_F16>(a, p, s);
}
}  // namespace mxq_kv
