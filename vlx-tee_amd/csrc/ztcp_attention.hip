// ztcp_attention.hip -- attention of new tokens over hot pages: the kernels of
// ztcp_attend.h where each token sees those in front of it and itself.
#include "ztcp_attend.h"

extern "C" size_t ztcp_paged_attention_workspace(const ztcp_paged_batch* batch, const ztcp_page_pool* pool,
                                                 const ztcp_geometry* g, int64_t q_heads) {
    return workspace_of(batch, pool, g, q_heads, false);
}

extern "C" int ztcp_paged_attention(const void* q, int64_t q_stride, void* out, float* lse, int64_t q_heads,
                                    const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g,
                                    float scale, void* workspace, size_t workspace_bytes, void* stream) {
    return attend<false>(q, q_stride, out, lse, q_heads, pool, batch, g, nullptr, 0, scale, workspace, workspace_bytes, stream);
}
