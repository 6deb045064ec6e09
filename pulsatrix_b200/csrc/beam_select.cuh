// Launch interface of the selection over beams and vocabulary (beam_select.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace psx {

constexpr int kMostKept = 128;         // candidates per group
constexpr int kMostSelectBeams = 64;

struct BeamPart {        // what is left of a part of a row
    double sum;          // of exp(logit - top) over the part
    float top;           // the part's largest logit; -inf: none
    int32_t not_finite;  // it holds a NaN or +inf
};

struct BeamEntry {
    float logit;
    int32_t token;
};

// x / by for x * by < 2^32, by a multiplication: the magic number is 2^32 / by rounded up, off by less than `by` 2^-32 of it.
struct Quotients {
    uint32_t one = 1, magic = 0;
    Quotients() = default;
    explicit Quotients(uint32_t by);
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t quotient(uint32_t x) const { return one ? x : __umulhi(x, magic); }
#endif
};

struct BeamSelectParams {
    const float* logits;      // (groups * beams, vocab), row r at logits + r * row_stride
    const float* scores;      // (groups * beams): the beams' scores so far
    const uint8_t* finished;  // (groups * beams) or null
    float* out_scores;        // (groups, keep)
    int64_t* parents;         // (groups, keep): the beam that a candidate continues, 0 .. beams - 1
    int64_t* tokens;          // (groups, keep)
    int32_t* group_status;    // (groups) or null
    int64_t groups, row_stride, finished_token;
    int32_t beams, vocab, keep;
    int32_t parts;            // of a row
    int32_t values;           // logits per thread of a chunk: 4 or 16
    int32_t chunks;           // of a part, 1 to 8
    Quotients by_parts, by_lists;  // the parts of a row, those of a group's rows together
    int32_t aligned;          // every row starts on a 16-byte boundary and is a multiple of four long
    int32_t* arrived;         // scratch: (groups), zero between calls
    BeamPart* part_stats;     // (groups * beams, parts)
    BeamEntry* entries;       // (groups * beams, parts, keep), best first
};

// parts, values, chunks and aligned, from the sizes and pointers.
void plan_beam_select(BeamSelectParams& p, int sm_count);
cudaError_t launch_beam_select(const BeamSelectParams& p, cudaStream_t stream);

}  // namespace psx
