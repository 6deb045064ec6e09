// Launch interface of the attention of whole prompts (prompt_attention.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace psx {

struct PromptAttentionParams {
    const void* q;  // (total_q, heads, head_dim), a position at q + i * q_stride elements; k and v likewise
    const void* k;  // (total_k, kv_heads, head_dim)
    const void* v;
    void* out;      // (total_q, heads, head_dim), contiguous
    const int64_t* q_offsets;  // (batch + 1): sequence b's queries are q_offsets[b] .. q_offsets[b + 1]
    const int64_t* k_offsets;
    int32_t* status;  // bit 0 is set when a bounded wait ran out; may be null
    void* split;      // scratch for fp32 operands, prompt_split_bytes()
    int64_t total_q, total_k, q_stride, k_stride, v_stride, window;
    uint64_t wait_limit_ns;
    int32_t batch, heads, kv_heads, head_dim, type, causal;
    uint32_t extra_bytes;  // announced beyond what the copies deliver: 0 (see psx_b200_test_short_copy)
    float scale;
};

size_t prompt_split_bytes(const PromptAttentionParams& p);
// *launches: kernels launched.  cudaErrorNotSupported: the driver does not know tensor maps.
cudaError_t launch_prompt_attention(const PromptAttentionParams& p, int sm_count, cudaStream_t stream, int* launches);

}  // namespace psx
