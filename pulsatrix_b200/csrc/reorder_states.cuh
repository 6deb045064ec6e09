// Launch interface of the rows of states that follow their beams (reorder_states.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace psx {

constexpr int kStatesPerLaunch = 64;  // (their descriptions travel in the launch's parameters)
constexpr int kMostBeams = 64;

struct BeamState {
    char* data;                   // (groups * beams, heads, positions) of position_bytes each
    int64_t heads, positions, position_bytes;
    int64_t tokens_per_position;  // a position holds what belongs to so many tokens
    int32_t splits;               // blocks that share the positions of a head
    int32_t first_block;          // of this state's blocks in the launch
    int32_t width;                // bytes that a thread moves at a time
};

template <int most>
struct ReorderParamsOf {
    BeamState states[most];
    int32_t count, beams;
    int64_t groups;
    const int64_t* parents;  // (groups, beams): row of the same group, else the row stays as it is
    const int64_t* lengths;  // (groups * beams): tokens that a row holds; null: all positions
};
using ReorderParams = ReorderParamsOf<kStatesPerLaunch>;

// Fills in splits, first_block and width of p.states[0 .. p.count) and launches.  cudaErrorInvalidValue: more than
// kMostBeams beams or too many blocks.
cudaError_t launch_reorder_states(ReorderParams& p, int sm_count, cudaStream_t stream);

}  // namespace psx
