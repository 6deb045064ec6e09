// Launch interface of the attention of new positions over a cache in pages (decode_attention_pages.cu).
#pragma once

#include "paged_cache.cuh"

namespace psx {

struct PagedAttentionParams {
    PagedCacheView cache;
    const void* q;   // (rows * q_len, heads, head_dim)
    void* context;   // like q
    float* partial;  // scratch: the pieces' contexts, maxima and sums
    int32_t* arrived;  // scratch: pieces of a (row, kv head) that are there, zero between calls
    int64_t window;
    int32_t heads, group, q_len;
    int32_t rows;    // query rows of a (row, kv head): group * q_len, 16 at most
    int32_t type, causal;
    int32_t row_groups;  // blocks beside one another that share these (beyond 128 dimensions, eight each)
    int32_t pieces;  // blocks of a (row, kv head)
    int32_t spread;  // of which so many fill the GPU
    float scale;
};

// row_groups, pieces and spread.
void plan_paged_attention(PagedAttentionParams& p, int sm_count);
size_t paged_attention_partial_bytes(const PagedAttentionParams& p);
int64_t paged_attention_counters(const PagedAttentionParams& p);
cudaError_t launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream);

}  // namespace psx
