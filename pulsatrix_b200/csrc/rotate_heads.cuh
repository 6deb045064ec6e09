// Launch interface of queries and keys on their way from a projection into the cache (rotate_heads.cu).
#pragma once

#include "paged_cache.cuh"

namespace psx {

struct RotateHeadsParams {
    const void *q, *k, *v;            // (total, heads or kv_heads, head_dim), a position at + i * stride elements
    void *q_out, *k_out;              // (total, heads or kv_heads, head_dim), contiguous; k_out may be null
    const void *q_weight, *k_weight;  // (head_dim) of the same type; null: no norm
    const double* frequencies;        // (rotated / 2)
    const int64_t *offsets, *first;   // (batch + 1), (batch)
    int32_t* row_status;              // (batch) or null
    int64_t total, q_stride, k_stride, v_stride;
    PagedCacheView cache;             // keys == nullptr: none
    int32_t batch, heads, kv_heads, head_dim, rotated, interleaved, type;
    float eps, inverse_dims;
    int32_t slabs, slab_rows;         // shares of a position's heads: how many, and heads of one
};

cudaError_t launch_rotate_heads(RotateHeadsParams& p, int sm_count, cudaStream_t stream);

}  // namespace psx
