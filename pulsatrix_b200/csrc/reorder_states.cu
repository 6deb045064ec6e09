// Rows of states that follow their beams, in place: row j of a group becomes what row parents[j] was.
//
// A permutation with repetitions cannot be done row by row in place; what makes it safe here is that a thread owns a column
// (the same few bytes of every row of a group): it reads all the parents' bytes that it needs into registers, then writes.
// No other thread touches that column, so there is no barrier, no second buffer and no order between blocks.  Rows that stay
// are neither read (unless another row comes from them) nor written, and what lies behind a row's length is not moved.
//
// Bound by HBM: each parent is read once (rows of one parent read the same bytes, the later reads come out of L1 or L2) and
// each changed row written once.  A thread has as many loads in flight as rows of its group change; 16 bytes each up to 16
// beams, 8 up to 32 and 4 up to 64, so that they take 64 registers at most.
#include "reorder_states.cuh"

#include <algorithm>
#include <type_traits>

namespace psx {
namespace {

constexpr int kThreads = 256;
constexpr int kFewStates = 8;  // a layer's or two layers' caches

struct Move {
    int64_t to, from, end;  // byte offsets of the two rows; bytes of a head that are taken over
};

template <int beams, class Bytes>
__device__ __forceinline__ void move_columns(char* base, int64_t begin, int64_t end, int64_t step, int moved, const volatile Move* moves) {
#pragma unroll 1
    for (int64_t at = begin; at < end; at += step) {
        Bytes held[beams];
#pragma unroll
        for (int k = 0; k < beams; ++k) {  // (volatile: the moves stay in shared memory, the registers are for the bytes)
            if (k < moved && at < moves[k].end) held[k] = *reinterpret_cast<const Bytes*>(base + moves[k].from + at);
        }
#pragma unroll
        for (int k = 0; k < beams; ++k) {
            if (k < moved && at < moves[k].end) *reinterpret_cast<Bytes*>(base + moves[k].to + at) = held[k];
        }
    }
}

template <int beams, int most>
__global__ void __launch_bounds__(kThreads) reorder_states_kernel(const __grid_constant__ ReorderParamsOf<most> p) {
    __shared__ Move moves[beams];
    __shared__ int count;
    __shared__ int64_t longest;
    int which = 0;
    while (which + 1 < p.count && (int)blockIdx.x >= p.states[which + 1].first_block) ++which;
    const BeamState& s = p.states[which];
    int64_t rest = (int)blockIdx.x - s.first_block;
    const int64_t split = rest % s.splits;
    rest /= s.splits;
    const int64_t head = rest % s.heads, group = rest / s.heads;
    const int64_t head_bytes = s.positions * s.position_bytes, row_bytes = s.heads * head_bytes;
    if (threadIdx.x < 32) {  // the rows that change, in order
        int found = 0;
        int64_t most = 0;
        for (int base = 0; base < p.beams; base += 32) {
            const int j = base + threadIdx.x;
            const int64_t parent = j < p.beams ? p.parents[group * p.beams + j] : -1;
            int64_t end = 0;
            if (parent >= 0 && parent < p.beams && parent != j) {
                int64_t positions = s.positions;
                if (p.lengths) {
                    const int64_t tokens = max(p.lengths[group * p.beams + parent], (int64_t)0);
                    positions = min(positions, tokens / s.tokens_per_position + (tokens % s.tokens_per_position != 0));
                }
                end = positions * s.position_bytes;
            }
            const unsigned changed = __ballot_sync(0xffffffffu, end > 0);
            if (end > 0) {
                const int at = found + __popc(changed & ((1u << threadIdx.x) - 1));
                moves[at] = {j * row_bytes, parent * row_bytes, end};
            }
            found += __popc(changed);
            most = max(most, end);
        }
        for (int step = 16; step > 0; step /= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, step));
        if (threadIdx.x == 0) count = found, longest = most;
    }
    __syncthreads();
    char* base = s.data + group * p.beams * row_bytes + head * head_bytes;
    const int64_t begin = (split * kThreads + threadIdx.x) * s.width, step = (int64_t)s.splits * kThreads * s.width;
    if constexpr (beams <= 16) {
        if (s.width == 16) return move_columns<beams, uint4>(base, begin, longest, step, count, moves);
    }
    if constexpr (beams <= 32) {
        if (s.width == 8) return move_columns<beams, uint2>(base, begin, longest, step, count, moves);
    }
    if (s.width == 4) return move_columns<beams, uint32_t>(base, begin, longest, step, count, moves);
    move_columns<beams, uint8_t>(base, begin, longest, step, count, moves);
}

}  // namespace

cudaError_t launch_reorder_states(ReorderParams& p, int sm_count, cudaStream_t stream) {
    if (p.beams > kMostBeams) return cudaErrorInvalidValue;
    int64_t heads = 0;
    for (int i = 0; i < p.count; ++i) heads += p.states[i].heads;
    // As many blocks as fill the GPU some three times over where the positions allow it: lengths are not known here, and blocks
    // that find little to do end early.
    const int64_t wanted = std::max<int64_t>(1, (int64_t)sm_count * 24 / std::max<int64_t>(1, heads * p.groups));
    int64_t blocks = 0;
    for (int i = 0; i < p.count; ++i) {
        BeamState& s = p.states[i];
        const uint64_t lies = reinterpret_cast<uint64_t>(s.data) | (uint64_t)s.position_bytes;
        const int widest = p.beams <= 16 ? 16 : p.beams <= 32 ? 8 : 4;
        s.width = lies % 16 == 0 ? 16 : lies % 8 == 0 ? 8 : lies % 4 == 0 ? 4 : 1;
        s.width = std::min(s.width, widest);
        const int64_t trips = (s.positions * s.position_bytes / s.width + kThreads - 1) / kThreads;
        s.splits = (int32_t)std::max<int64_t>(1, std::min({trips, wanted, (int64_t)65536}));
        s.first_block = (int32_t)blocks;
        blocks += p.groups * s.heads * s.splits;
        if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    }
    if (blocks == 0) return cudaSuccess;
    const auto launch = [&](const auto& params, auto few) {
        constexpr int most = decltype(few)::value;
        if (p.beams <= 4) reorder_states_kernel<4, most><<<(unsigned)blocks, kThreads, 0, stream>>>(params);
        else if (p.beams <= 8) reorder_states_kernel<8, most><<<(unsigned)blocks, kThreads, 0, stream>>>(params);
        else if (p.beams <= 16) reorder_states_kernel<16, most><<<(unsigned)blocks, kThreads, 0, stream>>>(params);
        else if (p.beams <= 32) reorder_states_kernel<32, most><<<(unsigned)blocks, kThreads, 0, stream>>>(params);
        else reorder_states_kernel<64, most><<<(unsigned)blocks, kThreads, 0, stream>>>(params);
    };
    if (p.count <= kFewStates) {  // (a launch copies its parameters: half a kilobyte instead of four)
        ReorderParamsOf<kFewStates> few;
        std::copy(p.states, p.states + p.count, few.states);
        few.count = p.count, few.beams = p.beams, few.groups = p.groups, few.parents = p.parents, few.lengths = p.lengths;
        launch(few, std::integral_constant<int, kFewStates>{});
    } else {
        launch(p, std::integral_constant<int, kStatesPerLaunch>{});
    }
    return cudaGetLastError();
}

}  // namespace psx
