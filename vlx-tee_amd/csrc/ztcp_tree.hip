// ztcp_tree.hip -- attention of drafted tokens that form a tree over hot pages:
// the kernels of ztcp_attend.h where each new token sees all tokens in front of
// the new ones and, of the new ones, those in its mask.
#include "ztcp_attend.h"

extern "C" size_t ztcp_tree_attention_workspace(const ztcp_paged_batch* batch, const ztcp_page_pool* pool,
                                                const ztcp_geometry* g, int64_t q_heads) {
    return workspace_of(batch, pool, g, q_heads, true);
}

extern "C" int ztcp_tree_attention(const void* q, int64_t q_stride, void* out, float* lse, int64_t q_heads,
                                   const ztcp_page_pool* pool, const ztcp_paged_batch* batch, const ztcp_geometry* g,
                                   const uint64_t* tree_mask, int64_t tree_words, float scale, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    return attend<true>(q, q_stride, out, lse, q_heads, pool, batch, g, tree_mask, tree_words, scale, workspace, workspace_bytes,
                        stream);
}
