// Sums of the counts of a batch's rows, taken by every block for itself: work that depends on lengths in device memory is
// shared out over the blocks without a launch that prepares it.
#pragma once

#include <stdint.h>

namespace psx {

constexpr int64_t kMostPrefixRows = 4096;  // (prefix[] is 16 KB of shared memory then)

// prefix[0] = 0, prefix[r + 1] = prefix[r] + count(r) for r < rows; `carry`: shared, one int per warp.  All
// threads of the block (whole warps, 32 at most) call it; the sums are readable by all of them afterwards.
template <class Count>
__device__ __forceinline__ void sum_of_rows(int rows, int* prefix, int* carry, Count count) {
    const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // Every thread takes neighbouring rows, so that the lengths of many rows are on their way at once.
    const int each = (rows + (int)blockDim.x - 1) / (int)blockDim.x, first = min((int)threadIdx.x * each, rows), end = min(first + each, rows);
    int mine = 0;
#pragma unroll 4
    for (int row = first; row < end; ++row) mine += count(row);
    int sum = mine;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, sum, step);
        if (lane >= step) sum += other;
    }
    if (lane == 31) carry[warp] = sum;
    __syncthreads();
    int before = sum - mine;
    for (int w = 0; w < warps; ++w) before += w < warp ? carry[w] : 0;
    if (threadIdx.x == 0) prefix[0] = 0;
    if (each == 1) {
        if (first < end) prefix[first + 1] = before + mine;
    } else {
#pragma unroll 4
        for (int row = first; row < end; ++row) {
            before += count(row);
            prefix[row + 1] = before;
        }
    }
    __syncthreads();
}

// The row whose share holds `item`: prefix[row] <= item < prefix[row + 1].
__device__ __forceinline__ int row_of_item(const int* prefix, int rows, int item) {
    int low = 0, high = rows - 1;
    while (low < high) {
        const int middle = (low + high) / 2;
        if (prefix[middle + 1] > item) high = middle;
        else low = middle + 1;
    }
    return low;
}

}  // namespace psx
