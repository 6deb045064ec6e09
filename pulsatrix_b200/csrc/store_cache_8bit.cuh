// A cache of keys and values in 8 bits, and the launch interface of its writer (store_cache_8bit.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace psx {

struct Cache8bitView {
    uint8_t* key_codes;    // (batch, kv_heads, max_len, head_dim) e4m3
    float* key_scales;     // (batch, kv_heads, blocks): a position's values are its codes times its block's scale
    uint8_t* value_codes;
    float* value_scales;
    int64_t batch, max_len, blocks;  // blocks = ceil(max_len / block)
    int32_t kv_heads, head_dim, block;
};

struct StoreCacheParams {
    Cache8bitView cache;
    const void* keys;        // (total, kv_heads, head_dim): the new positions of all rows, one row behind the other
    const void* values;
    const int64_t* offsets;  // (batch + 1): row b's new positions are offsets[b] .. offsets[b + 1]
    const int64_t* cached;   // (batch): positions that row b holds already
    int32_t* row_status;     // (batch) or null
    int64_t total, key_stride, value_stride;  // elements from one position to the next
    int32_t type;
};

constexpr int32_t kRowOk = 0, kRowCacheFull = 64, kRowBadOffsets = 65;

cudaError_t launch_store_cache_8bit(const StoreCacheParams& p, int sm_count, cudaStream_t stream);

}  // namespace psx
