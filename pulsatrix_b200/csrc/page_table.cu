// Bookkeeping of a cache in pages, on the device: room for new positions, rows that follow their beams, what is given back, and
// pools brought together.
//
// A row's positions lie in the pages that its entries name, and a page may be named by several rows: references counts the entries in
// use that do.  That count is all there is to know about a page; it is free where it is 0, so there is no list of free pages to keep, and
// which pages a row gets depends on the table alone: the lowest free ones, row after row.  A row that goes on in a last page which others
// hold too gets a page of its own and a copy of what it sees of the old one (the last of the rows that go on in it keeps it where nobody else
// holds it, unless that would write over what one of them holds that got no page).  So beams share their prompt's pages, and following a beam moves table entries, four bytes per page and row, instead of the
// cache.
//
// Bound by latency but for the copies, which run at HBM's rate (a thousand pages of 64 KB that move in four pools: 80 us, 6.7 TB/s).  One block gives pages out, and
// one pairs movers and free places, reading the references of a pool half of which is free: release and extension of 64 rows that ask for a page each take 10 us
// with 16,384 pages, 21 with 81,920 and 129 with a million, a plan of moves 10, 35 and 383; rows that ask for none 6 whatever the pool.  Rows that part are compared with
// all rows: 16 us for 512 of them, 460 for 4096, and 100 more where they are refused.
#include "page_table.cuh"

#include <algorithm>

#include "psx_device.cuh"

namespace psx {
namespace {

constexpr int kPlanThreads = 1024;  // of the one block that gives pages out
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kRowsPerThread = kMostPageRows / kPlanThreads;
constexpr int kRowOk = 0, kRowCacheFull = 64, kRowBad = 65;  // (psx_row_status)

// The sum of the values of the threads before this one; `total`: that of all.  `carry`: shared, one per warp; the block meets twice.
template <class T>
__device__ __forceinline__ T sum_before(T mine, T* carry, T& total) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    T sum = mine;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
        const T other = __shfl_up_sync(0xffffffffu, sum, step);
        if (lane >= step) sum += other;
    }
    if (lane == 31) carry[warp] = sum;
    __syncthreads();
    T before = sum - mine, all = lane < warps ? carry[lane] : T(0), up_to = all;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
        const T other = __shfl_up_sync(0xffffffffu, up_to, step);
        if (lane >= step) up_to += other;
    }
    total = __shfl_sync(0xffffffffu, up_to, 31);
    before += __shfl_sync(0xffffffffu, up_to - all, warp);
    __syncthreads();
    return before;
}

// Four references from `at` on; behind the last page: not free.
__device__ __forceinline__ int4 four_references(const PageTableView& t, int at) {
    if (at + 4 <= t.num_pages && reinterpret_cast<uintptr_t>(t.references) % 16 == 0) return __ldcg(reinterpret_cast<const int4*>(t.references + at));
    int4 r;
    r.x = at < t.num_pages ? __ldcg(t.references + at) : 1;
    r.y = at + 1 < t.num_pages ? __ldcg(t.references + at + 1) : 1;
    r.z = at + 2 < t.num_pages ? __ldcg(t.references + at + 2) : 1;
    r.w = at + 3 < t.num_pages ? __ldcg(t.references + at + 3) : 1;
    return r;
}

// ---- room for new positions ------------------------------------------------------------------------------------------------
// One block.  The references are read only where a page is asked for (one step in page_size for a row that grows by one position), once for
// the number of free pages, as far as they are asked for, and once to give them out.
__global__ void __launch_bounds__(kPlanThreads) extend_pages_kernel(const __grid_constant__ ExtendPagesParams p) {
    extern __shared__ __align__(16) char shared[];
    __shared__ uint64_t carry[kPlanWarps];
    const PageTableView& t = p.table;
    const int rows = t.rows;
    int* ends = reinterpret_cast<int*>(shared);  // pages that rows 0 .. row ask for together (more than there are: one more than those)
    int* goes_on = ends + (rows + 3) / 4 * 4;    // the shared page that a row goes on in; then only of those that copy it; else -1
    grid_dependency_wait();
    grid_dependents_may_launch();

    int status[kRowsPerThread], length[kRowsPerThread], added[kRowsPerThread], held_by[kRowsPerThread];
    const int each = (rows + kPlanThreads - 1) / kPlanThreads, first = min((int)threadIdx.x * each, rows), count = min(each, rows - first);
    bool shares = false;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        status[i] = kRowOk, length[i] = added[i] = held_by[i] = 0;
        if (i >= count) continue;
        const int row = first + i;
        const int64_t more = p.added[row], before = t.lengths[row];
        int page = -1;
        if (more < 0 || before < 0 || before > t.capacity()) {
            status[i] = kRowBad;
        } else if (more > t.capacity() - before) {
            status[i] = kRowCacheFull;
        } else {
            length[i] = (int)before, added[i] = (int)more;
            if (more > 0 && (length[i] & (t.page_size - 1)) != 0) {
                page = t.pages[(int64_t)row * t.max_pages + (length[i] >> t.shift)];
                if (!t.real(page)) status[i] = kRowBad, added[i] = 0, page = -1;
                else held_by[i] = __ldcg(t.references + page);
                if (held_by[i] <= 1) page = -1;
            }
        }
        shares |= page >= 0;
        goes_on[row] = page;
    }
    if (threadIdx.x < 4) goes_on[rows + threadIdx.x] = -1;
    bool copies[kRowsPerThread] = {}, keeps[kRowsPerThread] = {};
    if (__syncthreads_or(shares)) {
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            if (i >= count || goes_on[first + i] < 0) continue;
            const int page = goes_on[first + i];
            int going = 0, last = 0;
            for (int row = 0; row < (rows + 3) / 4 * 4; row += 4) {  // (behind the last row: -1)
                const int4 four = *reinterpret_cast<const int4*>(goes_on + row);
                if (four.x == page) ++going, last = row;
                if (four.y == page) ++going, last = row + 1;
                if (four.z == page) ++going, last = row + 2;
                if (four.w == page) ++going, last = row + 3;
            }
            keeps[i] = going == held_by[i] && last == first + i;
            copies[i] = !keeps[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            if (i < count && !copies[i]) goes_on[first + i] = -1;
        }
    }
    int64_t mine = 0;
    int need[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        need[i] = t.pages_of(length[i] + added[i]) - t.pages_of(length[i]) + copies[i];
        mine += need[i];
    }
    uint64_t all;
    int64_t before = (int64_t)sum_before((uint64_t)mine, carry, all);
    const int asked = (int)min((int64_t)all, (int64_t)t.num_pages + 1);
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        before += need[i];
        if (i < count) {
            ends[first + i] = (int)min(before, (int64_t)t.num_pages + 1);
            p.copies[first + i].filled = 0;
        }
    }
    int available = 0;
    if (asked > 0) {
        constexpr int kRead = 4;                               // of four references, of a thread at a time
        constexpr int kStretch = kRead * 4 * kPlanThreads;     // of pages
        int4 held[kRead];
        uint64_t ahead = 0, totals = 0;  // free pages before this thread's, and in all, of each of the four: 16 bits each
        const auto read = [&](int base) {
            uint64_t free = 0;
#pragma unroll
            for (int k = 0; k < kRead; ++k) {
                const int64_t at = (int64_t)base + (k * kPlanThreads + (int)threadIdx.x) * 4;
                held[k] = at < t.num_pages ? four_references(t, (int)at) : make_int4(1, 1, 1, 1);
                free |= (uint64_t)((held[k].x == 0) + (held[k].y == 0) + (held[k].z == 0) + (held[k].w == 0)) << (16 * k);
            }
            ahead = sum_before(free, carry, totals);
            return (int)((totals & 0xffff) + (totals >> 16 & 0xffff) + (totals >> 32 & 0xffff) + (totals >> 48));
        };
        int base = 0;
        for (; base < t.num_pages; base += kStretch) {
            available += read(base);
            if (available >= asked) break;
        }
        // Rows in order, until one asks for more than there is: the pages of those before it.
        int low = 0, high = rows;  // the first row whose end is beyond what is there
        while (low < high) {
            const int middle = (low + high) / 2;
            if (ends[middle] > available) high = middle;
            else low = middle + 1;
        }
        const int given = low > 0 ? ends[low - 1] : 0;
        int rank = 0;
        bool at_hand = base == 0;  // (the first stretch was enough, and is still there)
        for (base = 0; base < t.num_pages && rank < given; base += kStretch) {
            if (!at_hand) read(base);
            at_hand = false;
#pragma unroll
            for (int k = 0; k < kRead; ++k) {
                const int here[4] = {held[k].x == 0, held[k].y == 0, held[k].z == 0, held[k].w == 0};
                int next = rank + (int)(ahead >> (16 * k) & 0xffff);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (here[j] && next < given) {
                        const int page = base + (k * kPlanThreads + (int)threadIdx.x) * 4 + j;
                        int from = 0, to = rows - 1;  // the row that the page is for: the first that ends behind it
                        while (from < to) {
                            const int middle = (from + to) / 2;
                            if (ends[middle] > next) to = middle;
                            else from = middle + 1;
                        }
                        const int slot = next - (from > 0 ? ends[from - 1] : 0), length_of = (int)t.lengths[from], old = goes_on[from];
                        t.references[page] = 1;
                        const int entry = old >= 0 && slot == 0 ? length_of >> t.shift : t.pages_of(length_of) + slot - (old >= 0);
                        t.pages[(int64_t)from * t.max_pages + entry] = page;
                        if (old >= 0 && slot == 0) {
                            p.copies[from] = {old, page, length_of & (t.page_size - 1), 0};
                            atomicSub(t.references + old, 1);  // (another row holds it still: it does not become free meanwhile)
                        }
                    }
                    next += here[j];
                }
                rank += (int)(totals >> (16 * k) & 0xffff);
            }
        }
        // A row that would keep its page in place is refused like those before it where one of them, left in the page without a copy, holds more of it.
        if (available < asked) {
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i) {
                if (!keeps[i]) continue;
                const int page = t.pages[(int64_t)(first + i) * t.max_pages + (length[i] >> t.shift)], filled = length[i] & (t.page_size - 1);
                for (int row = 0; row < first + i; ++row) {
                    if (goes_on[row] == page && ends[row] > available && ((int)t.lengths[row] & (t.page_size - 1)) > filled) status[i] = kRowCacheFull;
                }
            }
        }
        __syncthreads();  // (lengths are read until here)
    }
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        if (i >= count) continue;
        if (need[i] > 0 && ends[first + i] > available) status[i] = kRowCacheFull;
        if (added[i] > 0 && status[i] == kRowOk) t.lengths[first + i] = length[i] + added[i];
        if (p.row_status) p.row_status[first + i] = status[i];
    }
}

// ---- copies of bytes ---------------------------------------------------------------------------------------------------------
constexpr int kCopyThreads = 256;

// `count` elements from one place to another; `each` are on their way per thread.
template <class Bytes>
__device__ __forceinline__ void copy_run(Bytes* to, const Bytes* from, int begin, int end) {
    constexpr int kAhead = 8;
    for (int at = begin + (int)threadIdx.x; at < end; at += kAhead * kCopyThreads) {
        Bytes held[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (at + k * kCopyThreads < end) held[k] = __ldcs(from + at + k * kCopyThreads);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (at + k * kCopyThreads < end) __stcs(to + at + k * kCopyThreads, held[k]);
        }
    }
}

__device__ __forceinline__ void copy_run(char* to, const char* from, int64_t begin, int64_t end, int width) {
    if (width == 16) copy_run(reinterpret_cast<uint4*>(to), reinterpret_cast<const uint4*>(from), (int)(begin / 16), (int)(end / 16));
    else if (width == 8) copy_run(reinterpret_cast<uint2*>(to), reinterpret_cast<const uint2*>(from), (int)(begin / 8), (int)(end / 8));
    else if (width == 4) copy_run(reinterpret_cast<uint32_t*>(to), reinterpret_cast<const uint32_t*>(from), (int)(begin / 4), (int)(end / 4));
    else copy_run(reinterpret_cast<uint8_t*>(to), reinterpret_cast<const uint8_t*>(from), (int)begin, (int)end);
}

struct CopyLastParams {
    PagePools pools;
    const PageCopy* copies;
    int32_t page_size, splits;  // blocks that share the heads of a (row, pool)
};

// A block per (row, pool, share of the heads): the head's filled positions are one run.
__global__ void __launch_bounds__(kCopyThreads) copy_last_pages_kernel(const __grid_constant__ CopyLastParams p) {
    grid_dependency_wait();
    const int split = blockIdx.x % p.splits, row = blockIdx.x / p.splits;
    const PageCopy copy = p.copies[row];
    if (copy.filled == 0) return;
    const PagePool& pool = p.pools.pool[blockIdx.y];
    const int64_t head_bytes = p.page_size * pool.position_bytes, page_bytes = pool.heads * head_bytes;
    for (int64_t head = split; head < pool.heads; head += p.splits) {
        copy_run(pool.data + copy.to * page_bytes + head * head_bytes, pool.data + copy.from * page_bytes + head * head_bytes, 0,
                 copy.filled * pool.position_bytes, pool.width);
    }
}

// ---- rows that follow their beams -------------------------------------------------------------------------------------------
// A block per group; a thread owns a column of the group's rows, the entries that name one page's worth of positions each: it reads all of
// them before it writes.  A page that a row held before and holds after is not counted.
constexpr int kForkThreads = 256, kForkColumns = 32 * kForkThreads;  // (entries in shared memory: fewer threads beyond 32 beams)

__global__ void __launch_bounds__(kForkThreads) fork_pages_kernel(const __grid_constant__ ForkPagesParams p) {
    extern __shared__ int column[];  // (beams, threads)
    __shared__ int length[kMostSharingBeams], parent[kMostSharingBeams];
    __shared__ int most;
    const PageTableView& t = p.table;
    const int threads = blockDim.x;
    grid_dependency_wait();
    grid_dependents_may_launch();
    const int64_t row0 = (int64_t)blockIdx.x * p.beams;
    if (threadIdx.x == 0) most = 0;
    __syncthreads();
    if ((int)threadIdx.x < p.beams) {
        const int j = threadIdx.x;
        const int64_t of = p.parents[row0 + j];
        length[j] = t.length((int)row0 + j);
        parent[j] = of >= 0 && of < p.beams ? (int)of : j;
        atomicMax(&most, t.pages_of(length[j]));
    }
    __syncthreads();
    for (int c = threadIdx.x; c < most; c += threads) {
        int32_t* at = t.pages + row0 * t.max_pages + c;
#pragma unroll 4
        for (int j = 0; j < p.beams; ++j) column[j * threads + threadIdx.x] = c < t.pages_of(length[j]) ? at[(int64_t)j * t.max_pages] : -1;
        for (int j = 0; j < p.beams; ++j) {
            if (parent[j] == j) continue;
            const int old = column[j * threads + threadIdx.x], now = column[parent[j] * threads + threadIdx.x];
            if (old == now) continue;
            if (t.real(now)) atomicAdd(t.references + now, 1);
            if (t.real(old)) atomicSub(t.references + old, 1);
            if (c < t.pages_of(length[parent[j]])) at[(int64_t)j * t.max_pages] = now;
        }
    }
    if ((int)threadIdx.x < p.beams && parent[threadIdx.x] != threadIdx.x) t.lengths[row0 + threadIdx.x] = length[parent[threadIdx.x]];
}

// ---- what is given back -----------------------------------------------------------------------------------------------------
constexpr int kReleaseThreads = 128;

__global__ void __launch_bounds__(kReleaseThreads) release_pages_kernel(const __grid_constant__ ReleasePagesParams p) {
    const PageTableView& t = p.table;
    grid_dependency_wait();
    grid_dependents_may_launch();
    const int row = blockIdx.x, length = t.length(row);
    const int kept = p.keep ? (int)min(max(p.keep[row], (int64_t)0), (int64_t)length) : 0;
    __syncthreads();  // (every thread has read the length)
    if (threadIdx.x == 0 && kept < length) t.lengths[row] = kept;
    for (int c = t.pages_of(kept) + threadIdx.x; c < t.pages_of(length); c += kReleaseThreads) {
        const int page = t.pages[(int64_t)row * t.max_pages + c];
        if (t.real(page)) atomicSub(t.references + page, 1);
    }
}

// ---- pools brought together -------------------------------------------------------------------------------------------------
// With `used` pages in use, those behind the first `used` places move into the free ones among them, both in ascending order.  No page is
// read and written, so the moves need no order.
__global__ void __launch_bounds__(kPlanThreads) compact_pages_kernel(const __grid_constant__ CompactPagesParams p) {
    __shared__ uint64_t carry[kPlanWarps];
    const PageTableView& t = p.table;
    grid_dependency_wait();
    grid_dependents_may_launch();
    int in_use = 0;
    for (int64_t at = threadIdx.x * 4; at < t.num_pages; at += 4 * kPlanThreads) {
        const int4 r = four_references(t, (int)at);
        in_use += (r.x > 0) + (r.y > 0 && at + 1 < t.num_pages) + (r.z > 0 && at + 2 < t.num_pages) + (r.w > 0 && at + 3 < t.num_pages);
    }
    uint64_t all;
    int64_t free_found = 0, moved = 0;
    sum_before((uint64_t)in_use, carry, all);
    const int64_t used = (int64_t)all;
    for (int64_t base = 0; base < t.num_pages; base += 4 * kPlanThreads) {
        const int64_t at = base + threadIdx.x * 4;
        const int4 r = at < t.num_pages ? four_references(t, (int)at) : make_int4(1, 1, 1, 1);
        const int held[4] = {r.x, r.y, r.z, r.w};
        uint64_t counts = 0, of_all;  // goals in the low half, movers in the high one
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at + k < used) counts += held[k] <= 0;
            else if (at + k < t.num_pages) counts += held[k] > 0 ? uint64_t(1) << 32 : 0;
        }
        const uint64_t before = sum_before(counts, carry, of_all);
        int64_t goal = free_found + (int64_t)(before & 0xffffffff), mover = moved + (int64_t)(before >> 32);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at + k < used) {
                if (held[k] <= 0) p.to[goal++] = (int)at + k;
            } else if (at + k < t.num_pages) {
                if (held[k] > 0) p.from[mover++] = (int)at + k;
            }
        }
        free_found += (int64_t)(of_all & 0xffffffff);
        moved += (int64_t)(of_all >> 32);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
        const int from = p.from[i], to = p.to[i];
        p.moved_to[from] = to;
        t.references[to] = t.references[from];
        t.references[from] = 0;
    }
    if (threadIdx.x == 0) {
        *p.used = used;
        *p.moves = (int)moved;
    }
}

struct MovePagesParams {
    CompactPagesParams plan;
    PagePools pools;
    int32_t entries;
};

constexpr int kPiece = 32768;  // bytes of a page that a block moves at a time

__global__ void __launch_bounds__(kCopyThreads) move_pages_kernel(const __grid_constant__ MovePagesParams p) {
    grid_dependency_wait();
    const PageTableView& t = p.plan.table;
    const int moves = *p.plan.moves;
    for (int i = 0; i < p.pools.count; ++i) {
        const PagePool& pool = p.pools.pool[i];
        const int64_t page_bytes = pool.heads * t.page_size * pool.position_bytes, pieces = (page_bytes + kPiece - 1) / kPiece;
        for (int64_t unit = blockIdx.x; unit < moves * pieces; unit += gridDim.x) {
            const int64_t move = unit / pieces, begin = unit % pieces * kPiece;
            copy_run(pool.data + p.plan.to[move] * page_bytes, pool.data + p.plan.from[move] * page_bytes, begin, min(begin + kPiece, page_bytes), pool.width);
        }
    }
    if (!p.entries) return;
    const int used = (int)*p.plan.used;
    for (int row = blockIdx.x; row < t.rows; row += gridDim.x) {
        const int count = t.pages_of(t.length(row));
        for (int c = threadIdx.x; c < count; c += kCopyThreads) {
            int32_t* at = t.pages + (int64_t)row * t.max_pages + c;
            const int page = *at;
            if (page >= used && page < t.num_pages) *at = p.plan.moved_to[page];
        }
    }
}

void set_widths(PagePools& pools) {
    for (int i = 0; i < pools.count; ++i) {
        const uint64_t lies = reinterpret_cast<uint64_t>(pools.pool[i].data) | (uint64_t)pools.pool[i].position_bytes;
        pools.pool[i].width = lies % 16 == 0 ? 16 : lies % 8 == 0 ? 8 : lies % 4 == 0 ? 4 : 1;
    }
}

}  // namespace

cudaError_t launch_extend_pages(const ExtendPagesParams& p, cudaStream_t stream) {
    return launch_overlapping(extend_pages_kernel, dim3(1), dim3(kPlanThreads), ((size_t)p.table.rows * 2 + 16) * sizeof(int), stream, p);
}

cudaError_t launch_copy_last_pages(const ExtendPagesParams& p, PagePools& pools, int sm_count, cudaStream_t stream) {
    set_widths(pools);
    int64_t heads = 1;
    for (int i = 0; i < pools.count; ++i) heads = std::max(heads, pools.pool[i].heads);
    CopyLastParams c;
    c.pools = pools;
    c.copies = p.copies;
    c.page_size = p.table.page_size;
    c.splits = (int)std::min<int64_t>(heads, std::max<int64_t>(1, (int64_t)sm_count * 16 / ((int64_t)p.table.rows * pools.count)));
    return launch_overlapping(copy_last_pages_kernel, dim3((unsigned)(p.table.rows * c.splits), (unsigned)pools.count), kCopyThreads, 0, stream, c);
}

cudaError_t launch_fork_pages(const ForkPagesParams& p, cudaStream_t stream) {
    const int threads = p.beams > kForkColumns / kForkThreads ? kForkThreads / 2 : kForkThreads;
    return launch_overlapping(fork_pages_kernel, dim3((unsigned)p.groups), dim3(threads), (size_t)p.beams * threads * sizeof(int), stream, p);
}

cudaError_t launch_release_pages(const ReleasePagesParams& p, cudaStream_t stream) {
    return launch_overlapping(release_pages_kernel, dim3((unsigned)p.table.rows), dim3(kReleaseThreads), 0, stream, p);
}

cudaError_t launch_compact_pages(const CompactPagesParams& p, cudaStream_t stream) {
    return launch_overlapping(compact_pages_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
}

cudaError_t launch_move_pages(const CompactPagesParams& p, PagePools& pools, bool entries, int sm_count, cudaStream_t stream) {
    set_widths(pools);
    MovePagesParams m;
    m.plan = p;
    m.pools = pools;
    m.entries = entries;
    return launch_overlapping(move_pages_kernel, dim3((unsigned)(sm_count * 8)), kCopyThreads, 0, stream, m);
}

}  // namespace psx
