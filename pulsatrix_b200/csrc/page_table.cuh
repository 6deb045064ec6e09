// Launch interface of the bookkeeping of a cache in pages (page_table.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace psx {

constexpr int kMostPageRows = 4096;   // (an extension holds 8 bytes of shared memory per row)
constexpr int kPoolsPerLaunch = 64;   // (their descriptions travel in the launch's parameters)
constexpr int kMostSharingBeams = 64;

// Rows of a page table hold positions 0 .. lengths[row] - 1, page_size of them in each of the pages that their first entries name.
struct PageTableView {
    int32_t* pages;       // (rows, max_pages)
    int64_t* lengths;     // (rows)
    int32_t* references;  // (num_pages): entries in use that name a page; 0: it is free
    int32_t rows, max_pages, num_pages;
    int32_t page_size, shift;  // a power of two and its logarithm

    __host__ __device__ int capacity() const { return max_pages * page_size; }  // (2^30 at most)
#ifdef __CUDACC__
    __device__ __forceinline__ int length(int row) const { return (int)min(max(lengths[row], (int64_t)0), (int64_t)capacity()); }
    __device__ __forceinline__ int pages_of(int length) const { return (length + page_size - 1) >> shift; }
    __device__ __forceinline__ bool real(int page) const { return (uint32_t)page < (uint32_t)num_pages; }
#endif
};

struct PagePool {
    char* data;  // (num_pages, heads, page_size) of position_bytes each
    int64_t heads, position_bytes;
    int32_t width;  // bytes that a thread moves at a time
};

struct PagePools {
    PagePool pool[kPoolsPerLaunch];
    int32_t count;
};

// A row whose last page was shared: its first `filled` positions go from page `from` to page `to`.
struct PageCopy {
    int32_t from, to, filled, unused;
};

struct ExtendPagesParams {
    PageTableView table;
    const int64_t* added;  // (rows): positions that the row is to hold more
    int32_t* row_status;   // (rows) or null
    PageCopy* copies;      // scratch: (rows)
};

struct ForkPagesParams {
    PageTableView table;
    const int64_t* parents;  // (groups, beams)
    int32_t groups, beams;
};

struct ReleasePagesParams {
    PageTableView table;
    const int64_t* keep;  // (rows) or null: nothing is kept
};

struct CompactPagesParams {
    PageTableView table;
    int64_t* used;  // device, 1: pages in use
    // scratch: pages that move and where they go, both ascending, (num_pages) each; where a page goes, (num_pages); how many move
    int32_t *from, *to, *moved_to, *moves;
};

inline size_t compact_scratch_bytes(int64_t num_pages) { return (size_t)(3 * num_pages + 1) * sizeof(int32_t); }

cudaError_t launch_extend_pages(const ExtendPagesParams& p, cudaStream_t stream);
cudaError_t launch_copy_last_pages(const ExtendPagesParams& p, PagePools& pools, int sm_count, cudaStream_t stream);  // (behind the former)
cudaError_t launch_fork_pages(const ForkPagesParams& p, cudaStream_t stream);
cudaError_t launch_release_pages(const ReleasePagesParams& p, cudaStream_t stream);
cudaError_t launch_compact_pages(const CompactPagesParams& p, cudaStream_t stream);
// The moves of the former in these pools; with `entries`, the table's too.
cudaError_t launch_move_pages(const CompactPagesParams& p, PagePools& pools, bool entries, int sm_count, cudaStream_t stream);

}  // namespace psx
