// Launch interface of the log-probabilities of given tokens (token_log_probs.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace psx {

constexpr int kMostTop = 128;  // alternatives of a row

struct TokenLogProbsParams {
    const void* logits;     // (rows, vocab), row r at + r * row_stride elements
    const int64_t* tokens;  // (rows) or null
    float* log_probs;       // (rows), with tokens
    float* entropy;         // (rows) or null
    float* top_log_probs;   // (rows, top), with top > 0
    int64_t* top_tokens;    // (rows, top)
    int32_t* row_status;    // (rows) or null
    int64_t rows, row_stride;
    int32_t vocab, top, type;
    int32_t parts;          // of a row, CTAs of a cluster: 1, 2, 4, 8 or 16
    int32_t chunks;         // of a part
    int32_t group;          // chunks whose largest logit a thread keeps as one
    int32_t vectors;        // of 16 bytes of a chunk, a thread's
};

// parts, chunks, group and vectors.
void plan_token_log_probs(TokenLogProbsParams& p, int sm_count);
cudaError_t launch_token_log_probs(const TokenLogProbsParams& p, cudaStream_t stream);

}  // namespace psx
