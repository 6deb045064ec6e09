// Launch interface of the log-probabilities of given tokens (token_log_probs.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace psx {

constexpr int kMostTop = 128;  // alternatives of a row

// What is left of a part of a row, m being its largest logit: over all of its logits but one that is m
struct LogProbPart {
    float top;       // m; -inf: none; NaN or +inf: a logit that is not finite
    float sum;       // of exp(x - m)
    float weighted;  // of (x - m) log2(e) exp(x - m), at most 0
    int32_t unused;
};

struct LogProbEntry {
    float logit;
    int32_t token;
};

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
    int32_t parts;          // of a row
    int32_t chunks;         // of a part, 1 to 8
    int32_t vectors;        // of 16 bytes of a chunk, a thread's
    int32_t* arrived;       // scratch: (rows), zero between calls
    LogProbPart* stats;     // scratch: (rows, parts)
    LogProbEntry* entries;  // scratch: (rows, parts, top), best first
};

// parts, chunks and vectors.
void plan_token_log_probs(TokenLogProbsParams& p, int sm_count);
cudaError_t launch_token_log_probs(const TokenLogProbsParams& p, cudaStream_t stream);

}  // namespace psx
