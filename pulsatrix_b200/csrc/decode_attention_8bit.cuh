// Launch interface of the attention over a cache held in 8 bits (decode_attention_8bit.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "store_cache_8bit.cuh"

namespace psx {

struct Attention8bitParams {
    Cache8bitView cache;
    const void* q;           // (batch, heads, q_len, head_dim)
    void* context;           // likewise
    const int64_t* lengths;  // (batch): positions of the cache that row b sees, the new ones among them
    float* partial;          // scratch: a piece per block of the launch
    int32_t* arrived;        // scratch: attention_8bit_counters(), zero between calls
    int64_t window;          // sliding window of a causal mask; 0: none
    int32_t heads, group, q_len, rows;  // rows = group * q_len
    int32_t type, causal;
    int32_t row_groups;      // of a kv head's query rows: blocks take eight beyond 128 dimensions
    int32_t pieces;          // blocks of every (row, kv head, group of query rows)
    int32_t spread;          // pieces that fill the GPU
    float scale;
};

void plan_attention_8bit(Attention8bitParams& p, int sm_count);  // row_groups, pieces and spread
int64_t attention_8bit_counters(const Attention8bitParams& p);
size_t attention_8bit_partial_bytes(const Attention8bitParams& p);
// cudaErrorInvalidValue: see psx_b200_decode_attention_8bit for the shapes that are taken.
cudaError_t launch_decode_attention_8bit(const Attention8bitParams& p, cudaStream_t stream);

}  // namespace psx
