// Attention of whole prompts, packed one behind the other: per sequence and head softmax(scale q k^T, masked) v, on the
// fifth-generation tensor cores, without the scores in memory.
//
// A CTA takes one or two tiles of 128 rows, queries of a sequence and of the heads that share a kv head, and goes through the keys that they see in blocks.  One thread
// asks for copies (tiled, 128-byte swizzle), one issues the products, and a warpgroup per tile turns scores into weights, a
// thread per query: it loads its row of scores from tensor memory, keeps the running maximum and sum in registers (no
// exchange between threads), and writes the weights back to tensor memory, in the place of the scores, from where they are the left
// operand of the second product.  The reference point of a row's weights moves only where its maximum has grown by more than 2^8
// (weights are then up to 2^8 times the first ones, which costs no precision).  fp16 weights start at 2^7, so that they use the type's range from
// 65,504 down: they have their 11 bits down to 2^-21 of the reference point's, and end at 2^-31 of it (from 1 on, those below 2^-25 were lost, and with
// them all of a context whose leading key has the value 0).
//
// 16-bit operands: two tiles, blocks of 128 keys, two stages of keys and of values (four up to 64 dimensions).  The first half of a block's
// weights is handed on while the second is made.  The context stays in tensor memory and is rescaled there when the reference point
// moves.  While the tensor core works for one tile the other tile's warpgroup works on its scores: the one issuing warp goes from
// tile to tile, which keeps the two half a turn apart (with an issuing warp for each, both tiles ask for the same unit at a time: 773 us
// instead of 662 for two prompts of up to 8192 positions, 32 heads of 128 in bf16, causal; 640 to 676 from box to box since).  Weights are rounded to the operands'
// type, an error of the size of the context's own rounding.
// Bound by a tile's turn: some 1700 clocks from scores to weights (570 for the maximum, 1024 of exponentials at four a clock and
// scheduler), 1024 of products, and the way between the two; 1.02 to 1.08 PFLOP/s at those sizes.  Tried and taken back: a share of the
// exponentials by a polynomial (no gain, 662 and 668 us), two threads for a query (771 us).
//
// Few groups of rows: where they would leave half of the SMs idle, the CTAs of a cluster, up to eight, take a piece of a group's keys each,
// leave their contexts, reference points and sums in their own shared memory and join them there, each its share of the rows, out of
// all of the others' (one head of 4096 positions of 128: 25 us instead of 61; fp32 50 instead of 134; 16 queries of 8 heads behind 16,000
// keys: 35 instead of 189).  The same through memory, the last CTA to end joining all: 33, 55 and 47 us.  Clusters of two where the GPU
// is between half full and twice full cost more than they gain (16 heads of 4096: 108 us instead of 70): most of them would be the
// short rows', and a CTA that finds nothing to do still takes its turn.
//
// fp32 operands: every number is split into three bf16 parts that add up to it (8 bits of the fraction each), and a product is the
// six products of parts that reach fp32's precision, the small ones first.  The keys' and values' parts are written by a kernel ahead,
// the queries' go into tensor memory once, the weights' as they are made.  One tile, blocks of 64 keys; the scores have two places,
// so that the next block's scores are formed while this block's weights are.  The tensor core cuts its sums off instead of rounding them, which
// adds up over thousands of keys; so a block's context is formed from zero and added up in registers (error of the context against
// 64 bits 2e-7, summed by the tensor core 5e-6).  Six bf16 products are still several times faster than the FP32 pipes.
// Bound by the products: 48 of 128 x 64 x 16 for the scores of a block and 128 dimensions (59 clocks each, the queries out of tensor
// memory), 24 of 128 x 128 x 16 for its context (64 clocks).  Blocks of 128 keys with the queries in shared memory need fewer clocks of the
// tensor core but all of shared memory's: 226 us instead of 221 for five prompts of up to 1501 positions with a prefix, 16 heads of 96.
//
// Rows behind a sequence's last key in a block belong to other sequences: their scores are masked, and their values are set to zero in
// shared memory, so that a NaN there is not seen here.
#include "prompt_attention.cuh"

#include <algorithm>

#include "elements.cuh"
#include "once_per_device.hpp"
#include "row_prefix.cuh"
#include "tensor_core.cuh"

namespace psx {
namespace {

constexpr float kNone = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileRows = 128;
constexpr int kMostPieces = 8;         // of a group of rows' keys, where there are few groups: the CTAs of a cluster
constexpr int kLeastShared = 5;        // blocks of keys that are shared out
constexpr float kMostGrowth = 8.0f;  // of a row's maximum, in powers of two, before its context is rescaled
constexpr float kHalfLift = 7.0f;    // fp16 weights are 2^7 at the reference point, 2^15 at most

template <int dims_, int parts_>
struct Shape {
    static constexpr int dims = dims_, parts = parts_;  // the head dimension, rounded up to 64 or 128
    static constexpr int tiles = parts == 1 ? 2 : 1;
    static constexpr int block = parts == 1 ? 128 : 64;
    static constexpr int stages = dims == 64 ? 4 : 2;
    static constexpr int threads = tiles * 128 + (parts == 1 ? 128 : 96);  // the warpgroups; copying, issuing, clearing (and an idle) warp
    static constexpr int slabs = dims / 64;            // a tile lies in slabs of 64 columns, rows of 128 bytes
    static constexpr int q_bytes = parts == 1 ? kTileRows * dims * 2 : 0;  // of a tile (fp32: in tensor memory)
    static constexpr int k_part = block * dims * 2, k_bytes = parts * k_part;  // (of the values too)
    static constexpr int shared = tiles * q_bytes + 2 * stages * k_bytes;
    // Columns of tensor memory: scores, whose places the weights take; what has no room there of fp32 weights; contexts; fp32 queries.
    static constexpr int score_places = parts == 1 ? tiles : 2;
    static constexpr int third_at = score_places * block, context_at = parts == 1 ? third_at : third_at + block / 2;
    static constexpr int query_at = context_at + tiles * dims, query_part = dims / 2;
    static_assert(query_at + (parts == 1 ? 0 : parts * query_part) <= 512);
    // A piece's result in shared memory, in floats: per tile (four dimensions, row) fours of the context, then a row's reference point and sum.
    static constexpr int tile_floats = kTileRows * (dims + 2);
    static_assert(tiles * tile_floats * 4 <= shared);
    // Column of a part of the weights that take the scores' place.
    static __host__ __device__ constexpr int weight_at(int place, int part) { return part == 2 ? third_at : place * block + part * (block / 2); }
};

struct alignas(64) PromptLaunch {
    CUtensorMap q_map, k_map, v_map;
    PromptAttentionParams p;
    int32_t steps;  // of 16 dimensions
    int32_t pieces;  // CTAs of a cluster
    int32_t packed, positions;  // heads, and positions, of a tile's rows
    int32_t dims16;  // the head dimension, rounded up to 16
};

// What a tile of queries sees: key j where first(i) <= j < end(i), i the query's number in its sequence.
struct Sight {
    int64_t keys, ahead;  // keys of the sequence; keys before the first query's own position
    int64_t window;
    bool causal;
    __device__ __forceinline__ int64_t end(int64_t i) const { return causal ? min(keys, i + ahead + 1) : keys; }
    __device__ __forceinline__ int64_t first(int64_t i) const { return causal && window > 0 ? max(i + ahead + 1 - window, (int64_t)0) : 0; }
};

__device__ __forceinline__ uint32_t pack(float low, float high, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}
__device__ __forceinline__ uint32_t pack(float low, float high, __half) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}

// All threads of the cluster's CTAs meet, each by itself.
__device__ __forceinline__ void cluster_meets() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// From the shared memory of the cluster's CTA `rank`, where this CTA has `address`.
template <class T>
__device__ __forceinline__ T load_of_peer(uint32_t address, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(address), "r"(rank));
    T x;
    if constexpr (sizeof(T) == 16) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
    else asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
    return x;
}

// Two floats as three bf16 pairs that add up to them, the largest part first.  What is left of a number after a part is exact; of
// one that is not finite it is 0, and the largest floats' first part is rounded down instead of to infinity.
__device__ __forceinline__ void split_pair(float low, float high, uint32_t& first, uint32_t& second, uint32_t& third) {
    const float largest = 3.3895313892515355e38f;  // of bf16
    const auto bounded = [&](float x) { return fabsf(x) < -kNone ? fminf(fmaxf(x, -largest), largest) : x; };
    first = pack(bounded(low), bounded(high), __nv_bfloat16{});
    const auto left = [](float x, uint32_t taken) { return fabsf(x) < -kNone ? x - __uint_as_float(taken) : 0.0f; };
    low = left(low, first << 16), high = left(high, first & 0xffff0000u);
    second = pack(low, high, __nv_bfloat16{});
    low -= __uint_as_float(second << 16), high -= __uint_as_float(second & 0xffff0000u);
    third = pack(low, high, __nv_bfloat16{});
}

// The same for numbers that are neither large nor infinite.
__device__ __forceinline__ void split_weights(float2 w, uint32_t& first, uint32_t& second, uint32_t& third) {
    first = pack(w.x, w.y, __nv_bfloat16{});
    w.x -= __uint_as_float(first << 16), w.y -= __uint_as_float(first & 0xffff0000u);
    second = pack(w.x, w.y, __nv_bfloat16{});
    w.x -= __uint_as_float(second << 16), w.y -= __uint_as_float(second & 0xffff0000u);
    third = pack(w.x, w.y, __nv_bfloat16{});
}

// {a, b} * {x, y} + {u, v}, each rounded as alone.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 x, float2 u) {
    float2 r;
    asm("{\n\t.reg .b64 a, x, u;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmov.b64 u, {%6, %7};\n\tfma.rn.f32x2 a, a, x, u;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(x.x), "f"(x.y), "f"(u.x), "f"(u.y));
    return r;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 x) {
    float2 r;
    asm("{\n\t.reg .b64 a, x;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tadd.rn.f32x2 a, a, x;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(x.x), "f"(x.y));
    return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Elem: the type of the products' operands (bf16 for the parts of fp32); Out: the type of the context; pieced: the CTAs of a cluster
// share a group of rows' keys.
template <class Elem, class Out, class S, bool pieced>
__global__ void __launch_bounds__(S::threads, 1) prompt_attention_kernel(const __grid_constant__ PromptLaunch launch) {
    extern __shared__ uint8_t raw_shared[];
    __shared__ uint64_t q_full, k_full[S::stages], v_full[S::stages], k_empty[S::stages], v_empty[S::stages];
    __shared__ uint64_t score_full[2], weight_full[2][2], context_full[2], ragged_there, cleared, drained;
    __shared__ uint32_t tensor_at;
    __shared__ uint32_t give_up;
    __shared__ int carry[32];
    const PromptAttentionParams& p = launch.p;
    uint8_t* shared = raw_shared + ((1024 - (smem_address(raw_shared) & 1023)) & 1023);
    int* prefix = reinterpret_cast<int*>(shared + S::shared);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    constexpr int kCopyWarp = S::tiles * 4, kIssueWarp = kCopyWarp + 1, kTailWarp = kCopyWarp + 2;
    constexpr int kRows = S::tiles * kTileRows;
    const int positions = S::tiles * launch.positions;  // of a CTA

    const auto queries_of = [&](int b) { return max(min(p.q_offsets[b + 1], p.total_q) - max(p.q_offsets[b], (int64_t)0), (int64_t)0); };
    sum_of_rows(p.batch, prefix, carry, [&](int b) { return (int)((queries_of(b) + positions - 1) / positions); });
    const int item = pieced ? blockIdx.x / launch.pieces : blockIdx.x, number = pieced ? blockIdx.x % launch.pieces : 0;
    const int units = p.heads / launch.packed, group_of_rows = item / units, head0 = item % units * launch.packed;
    if (group_of_rows >= prefix[p.batch]) return;
    const int b = row_of_item(prefix, p.batch, group_of_rows);
    const int64_t queries = queries_of(b), q_begin = max(p.q_offsets[b], (int64_t)0), k_begin = max(p.k_offsets[b], (int64_t)0);
    const int64_t keys = max(min(p.k_offsets[b + 1], p.total_k) - k_begin, (int64_t)0);
    const Sight sight{keys, keys - queries, p.window, p.causal != 0};
    // The last queries see the most keys: they come first, so that the short work is left for the end.
    const int64_t row0 = (int64_t)(prefix[b + 1] - 1 - group_of_rows) * positions;  // (in positions)
    if (row0 < 0 || row0 >= queries) return;  // (offsets that make no sense)
    int64_t ends[S::tiles];
    int64_t begin = sight.first(row0) / S::block;  // blocks of keys, for all tiles
    int counts[S::tiles], most = 0;
#pragma unroll
    for (int t = 0; t < S::tiles; ++t) {
        const int64_t first_row = row0 + t * launch.positions, last_row = min(first_row + launch.positions, queries) - 1;
        ends[t] = last_row < first_row ? 0 : max(sight.end(last_row), (int64_t)0);
        counts[t] = (int)max((ends[t] + S::block - 1) / S::block - begin, (int64_t)0);
        most = max(most, counts[t]);
    }
    int pieces = 1;
    if constexpr (pieced) {  // this CTA's piece of the blocks
        const int share = most < kLeastShared ? max(most, 1) : (most + launch.pieces - 1) / launch.pieces, before = number * share;
        pieces = max((most + share - 1) / share, 1);
        if (number >= pieces) {
            if (pieces > 1) cluster_meets(), cluster_meets();
            return;
        }
        begin += before;
        most = min(most - before, share);
#pragma unroll
        for (int t = 0; t < S::tiles; ++t) counts[t] = min(max(counts[t] - before, 0), share);
    }

    // The block that ends behind the sequence's last key, if there is one.
    const int ragged = most > 0 && (begin + most) * S::block > keys ? most - 1 : -1;

    if (threadIdx.x == 0) {
        barrier_init(&q_full, S::parts == 1 ? 1 : 128);
        for (int s = 0; s < S::stages; ++s) {
            barrier_init(&k_full[s], 1);
            barrier_init(&v_full[s], 1);
            barrier_init(&k_empty[s], 1);
            barrier_init(&v_empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            barrier_init(&score_full[t], 1);
            barrier_init(&weight_full[t][0], 128);
            barrier_init(&weight_full[t][1], 128);
            barrier_init(&context_full[t], 1);
        }
        barrier_init(&ragged_there, 1);
        barrier_init(&cleared, 1);
        barrier_init(&drained, 1);
        barrier_init_fence();
        give_up = 0;
    }
    if (warp == kIssueWarp) tensor_allocate(&tensor_at, 512);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = tensor_at;
    // The limit is that of a block's step; `blocks`: how many of them may lie between.
    const auto wait_alone = [&](uint64_t* bar, uint32_t parity, uint32_t blocks = 1) {
        const uint64_t limit = p.wait_limit_ns < ~0ull >> 32 ? p.wait_limit_ns * blocks : p.wait_limit_ns;
        if (barrier_wait_bounded(bar, parity, limit, &give_up)) return true;
        *(volatile uint32_t*)&give_up = 1;
        return false;
    };
    const auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t blocks = 1) {  // (a warp goes on as a whole or not at all)
        if (__all_sync(0xffffffffu, barrier_passed(bar, parity))) return true;
        return __all_sync(0xffffffffu, wait_alone(bar, parity, blocks)) != 0;
    };
    const uint32_t q_at = smem_address(shared), k_at = q_at + S::tiles * S::q_bytes, v_at = k_at + S::stages * S::k_bytes;

    // Of the registers that the CTA was launched with (168 a thread) the warpgroups with a row per thread get more: 2 * 224 + 56 = 3 * 168.
    const auto few_registers = [] {
        if constexpr (S::parts == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    };
    const auto many_registers = [] {
        if constexpr (S::parts == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    };

    if (warp == kCopyWarp) {
        few_registers();
        if (lane == 0 && most > 0) {
            const int kv_head = head0 / (p.heads / p.kv_heads);
            const auto fetch = [&](uint32_t to, int rows, const CUtensorMap* map, int y, int64_t z, int64_t total, uint64_t* bar) {
                for (int part = 0; part < S::parts; ++part) {
                    for (int slab = 0; slab < S::slabs; ++slab) {
                        if (slab * 64 >= p.head_dim) continue;
                        tiled_copy_to_shared(to + (part * S::slabs + slab) * rows * 128, map, slab * 64, y, (int)(part * total + z), bar);
                    }
                }
            };
            const uint32_t filled = (uint32_t)min(S::slabs, (p.head_dim + 63) / 64) * 128 * S::parts;  // bytes per row that arrive
            if constexpr (S::parts == 1) {
                uint32_t q_bytes = 0;
                for (int t = 0; t < S::tiles; ++t) q_bytes += counts[t] > 0 ? launch.positions * launch.packed * filled : 0;
                barrier_expect_bytes(&q_full, q_bytes);
                for (int t = 0; t < S::tiles; ++t) {
                    if (counts[t] > 0) fetch(q_at + t * S::q_bytes, kTileRows, &launch.q_map, head0, q_begin + row0 + t * launch.positions, p.total_q, &q_full);
                }
            }
            int asked = 0;
            bool fine = true;
            for (; asked < most; ++asked) {
                const int s = asked % S::stages, round = asked / S::stages;
                const int64_t z = k_begin + (begin + asked) * S::block;
                if (round > 0 && !(fine = wait_alone(&k_empty[s], (round - 1) & 1))) break;
                barrier_expect_bytes(&k_full[s], S::block * filled + p.extra_bytes);
                fetch(k_at + s * S::k_bytes, S::block, &launch.k_map, kv_head, z, p.total_k, &k_full[s]);
                if (round > 0 && !(fine = wait_alone(&v_empty[s], (round - 1) & 1))) {
                    barrier_wait_bounded(&k_full[s], round & 1, p.wait_limit_ns);
                    break;
                }
                barrier_expect_bytes(&v_full[s], S::block * filled);
                fetch(v_at + s * S::k_bytes, S::block, &launch.v_map, kv_head, z, p.total_k, &v_full[s]);
            }
            // Nothing is on its way into shared memory when the CTA ends.  (Without a failure every copy has been waited for.)
            if (*(volatile uint32_t*)&give_up || !fine) {
                if constexpr (S::parts == 1) barrier_wait_bounded(&q_full, 0, p.wait_limit_ns);
                for (int i = max(asked - S::stages, 0); i < asked; ++i) {
                    barrier_wait_bounded(&k_full[i % S::stages], (i / S::stages) & 1, p.wait_limit_ns);
                    barrier_wait_bounded(&v_full[i % S::stages], (i / S::stages) & 1, p.wait_limit_ns);
                }
            }
        }
    } else if (warp == kIssueWarp) {
        few_registers();
        // The warp waits as a whole, and meets after one thread has issued: lanes that went ahead to the next wait would hold it up.
        constexpr bool bfloat = __is_same(Elem, __nv_bfloat16);
        const uint32_t score_kind = product_descriptor(bfloat, false, kTileRows, S::block);
        const uint32_t context_kind = product_descriptor(bfloat, true, kTileRows, launch.dims16);
        // A descriptor's start address counts in 16 bytes, in its lowest bits.
        const uint64_t q_rows = operand_descriptor(q_at, 16, 1024), k_rows = operand_descriptor(k_at, 16, 1024);
        const uint64_t v_rows = operand_descriptor(v_at, S::block * 128, 1024);
        const auto score = [&](int t, int s, int place) {  // S = Q K^T of a tile and a stage of keys
            bool add = false;
            for (int sum = S::parts - 1; sum >= 0; --sum) {  // (the smallest products first)
                for (int part = 0; part <= sum; ++part) {
                    const uint64_t k = k_rows + ((s * S::k_bytes + (sum - part) * S::k_part) >> 4);
#pragma unroll
                    for (int step = 0; step < S::dims / 16; ++step) {
                        if (step >= launch.steps) break;
                        const uint64_t c = k + ((step / 4 * (S::block * 128) + step % 4 * 32) >> 4);
                        if constexpr (S::parts == 1) {
                            product_of_shared(tensor + place, q_rows + ((t * S::q_bytes + step / 4 * (kTileRows * 128) + step % 4 * 32) >> 4), c, score_kind, add);
                        } else {
                            product_of_tensor(tensor + place, tensor + S::query_at + part * S::query_part + step * 8, c, score_kind, add);
                        }
                        add = true;
                    }
                }
            }
        };
        const auto weigh = [&](int t, int place, int s, int from, int to, bool add) {  // O += P V, of the block's keys 16 from .. 16 to
            for (int sum = S::parts - 1; sum >= 0; --sum) {
                for (int part = 0; part <= sum; ++part) {
                    const uint64_t v = v_rows + ((s * S::k_bytes + (sum - part) * S::k_part) >> 4);
#pragma unroll
                    for (int step = from; step < to; ++step) {
                        product_of_tensor(tensor + S::context_at + t * S::dims, tensor + S::weight_at(place, part) + step * 8, v + (step * (16 * 128) >> 4),
                                          context_kind, add);
                        add = true;
                    }
                }
            }
        };
        const auto issue = [&](auto what) {
            if (elected()) what();
            __syncwarp();
        };
        const auto stage_wait = [&](uint64_t* full, int c) { return wait(&full[c % S::stages], (c / S::stages) & 1); };
        // The values of block c: the last one's when another warp has cleared what lies behind the sequence.
        const auto values_wait = [&](int c) {
            if (!stage_wait(v_full, c)) return false;
            if (c != ragged) return true;
            if (lane == 0) barrier_arrive(&ragged_there);
            return wait(&cleared, 0);
        };
        const auto last_tile = [&](int c) { return S::tiles == 2 && counts[S::tiles - 1] > c ? 1 : 0; };  // that works on block c
        bool fine = most == 0 || (wait(&q_full, 0) && stage_wait(k_full, 0));
        if (most > 0 && fine) {
            tensor_fence_after();
            if constexpr (S::tiles == 2) {
                for (int t = 0; t < 2; ++t) {
                    if (counts[t] == 0) continue;
                    issue([&] {
                        score(t, 0, t * S::block);
                        products_arrive(&score_full[t]);
                        if (t == last_tile(0)) products_arrive(&k_empty[0]);
                    });
                }
                for (int c = 0; c < most && fine; ++c) {
                    // What can be waited for while the weights are being made comes first.
                    fine = values_wait(c) && (c + 1 == most || stage_wait(k_full, c + 1));
                    for (int t = 0; t < 2 && fine; ++t) {
                        if (c >= counts[t]) continue;
                        fine = wait(&weight_full[t][0], c & 1);
                        if (!fine) break;
                        tensor_fence_after();
                        issue([&] { weigh(t, t, c % S::stages, 0, S::block / 32, c > 0); });
                        fine = wait(&weight_full[t][1], c & 1);  // (the second half's weights are still on their way)
                        if (!fine) break;
                        tensor_fence_after();
                        issue([&] {
                            weigh(t, t, c % S::stages, S::block / 32, S::block / 16, true);
                            if (c + 1 < counts[t]) {
                                score(t, (c + 1) % S::stages, t * S::block);
                                products_arrive(&score_full[t]);
                                if (t == last_tile(c + 1)) products_arrive(&k_empty[(c + 1) % S::stages]);
                            } else {
                                products_arrive(&context_full[t]);
                            }
                            if (t == last_tile(c)) products_arrive(&v_empty[c % S::stages]);
                        });
                    }
                }
            } else {
                issue([&] {
                    score(0, 0, 0);
                    products_arrive(&score_full[0]);
                    products_arrive(&k_empty[0]);
                });
                for (int c = 0; c < most && fine; ++c) {
                    if (c + 1 < most) {  // (in the place of block c - 1's weights, which the products before this one read)
                        fine = stage_wait(k_full, c + 1);
                        if (!fine) break;
                        issue([&] {
                            score(0, (c + 1) % S::stages, ((c + 1) & 1) * S::block);
                            products_arrive(&score_full[(c + 1) & 1]);
                            products_arrive(&k_empty[(c + 1) % S::stages]);
                        });
                    }
                    fine = values_wait(c) && wait(&weight_full[0][0], c & 1);
                    if (!fine) break;
                    tensor_fence_after();
                    issue([&] {
                        weigh(0, c & 1, c % S::stages, 0, S::block / 16, false);
                        products_arrive(&context_full[0]);
                        products_arrive(&v_empty[c % S::stages]);
                    });
                }
            }
        }
        // Every product has ended before tensor memory is given back.
        issue([&] { products_arrive(&drained); });
        barrier_wait_bounded(&drained, 0, p.wait_limit_ns);
    } else if (warp == kTailWarp) {
        few_registers();
        // Values behind the sequence's last key become zeros when their block has arrived.  (The issuing thread says when: it is the
        // one that follows the barriers' phases.)
        if (ragged >= 0) {
            const int s = ragged % S::stages;
            if (wait(&ragged_there, 0, most + 1)) {
                const int real = (int)(keys - (begin + ragged) * S::block), rows = S::block - real;
                for (int slab = 0; slab < S::parts * S::slabs; ++slab) {
                    uint4* row = reinterpret_cast<uint4*>(shared + (v_at - q_at) + s * S::k_bytes + slab * (S::block * 128) + real * 128);
                    for (int i = lane; i < rows * 8; i += 32) row[i] = make_uint4(0, 0, 0, 0);
                }
                shared_writes_before_async();
                __syncwarp();
                if (lane == 0) barrier_arrive(&cleared);
            }
        }
    } else if (warp < S::tiles * 4) {
        many_registers();
        const int t = warp / 4;
        // A tile's rows: positions, and of each the packed heads.  This thread's query; whether there is one.
        const int tile_row = (warp % 4) * 32 + lane;
        const auto row_of = [&](int tile, int r) { return row0 + tile * launch.positions + r / launch.packed; };
        const auto is_row = [&](int r, int64_t its) { return r < launch.positions * launch.packed && its < queries; };
        const int64_t row = row_of(t, tile_row);
        const int head = head0 + tile_row % launch.packed;
        const bool real = is_row(tile_row, row);
        const uint32_t lanes = tensor + ((uint32_t)(warp % 4) << 21);        // (32 lanes further: bits 16 up)
        const uint32_t context_at = lanes + S::context_at + t * S::dims;
        const int64_t end = sight.end(row), first = sight.first(row);
        // What all queries of the warp see needs no mask.
        const int64_t all_end = sight.end(row_of(t, tile_row - lane)), all_first = sight.first(min(row_of(t, tile_row - lane + 31), max(queries - 1, (int64_t)0)));
        const int count = counts[t];
        const float scale = p.scale * kLog2e;
        const float factor = fabsf(scale) < 1e-37f ? copysignf(1e-37f, scale) : scale;  // (masked scores times it stay infinite)
        const bool turned = factor < 0.0f;  // the lowest score weighs most
        const float masked = turned ? -kNone : kNone;
        float top = masked, total = 0.0f;   // of the scores before the factor
        bool fine = true;
        // fp32: the context is summed up here, a block's at a time.
        constexpr int kSums = S::parts == 1 ? 1 : S::dims;
        float context[kSums];
        const auto add_block = [&]() {
            if constexpr (S::parts == 3) {
#pragma unroll
                for (int i = 0; i < S::dims; i += 64) {
                    if (i >= launch.dims16) break;
                    float o[64];
                    tensor_load32(context_at + i, o);
                    tensor_load32(context_at + i + 32, o + 32);
                    tensor_loads_done();
#pragma unroll
                    for (int k = 0; k < 64; k += 2) {
                        const float2 sum = add_pair(make_float2(context[i + k], context[i + k + 1]), make_float2(o[k], o[k + 1]));
                        context[i + k] = sum.x, context[i + k + 1] = sum.y;
                    }
                }
            }
        };
        if constexpr (S::parts == 3) {  // the query's parts into tensor memory
#pragma unroll
            for (int i = 0; i < kSums; ++i) context[i] = 0.0f;
            if (count > 0) {
                const float* q = static_cast<const float*>(p.q) + (q_begin + row) * p.q_stride + (int64_t)head * p.head_dim;
#pragma unroll 1
                for (int i = 0; i < launch.dims16; i += 32) {
                    uint32_t packed[3][16];
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (real && i + k < p.head_dim) x = __ldg(reinterpret_cast<const float4*>(q + i + k));
                        split_pair(x.x, x.y, packed[0][k / 2], packed[1][k / 2], packed[2][k / 2]);
                        split_pair(x.z, x.w, packed[0][k / 2 + 1], packed[1][k / 2 + 1], packed[2][k / 2 + 1]);
                    }
#pragma unroll
                    for (int part = 0; part < 3; ++part) tensor_store16(lanes + S::query_at + part * S::query_part + i / 2, packed[part]);
                }
                tensor_stores_done();
                tensor_fence_before();
                barrier_arrive(&q_full);
            }
        }
        for (int c = 0; c < count; ++c) {
            const int place = S::tiles == 2 ? t : c & 1;
            fine = wait(&score_full[place], S::tiles == 2 ? c & 1 : (c / 2) & 1);
            if (!fine) break;
            tensor_fence_after();
            float x[S::block];
#pragma unroll
            for (int i = 0; i < S::block; i += 32) tensor_load32(lanes + place * S::block + i, x + i);
            tensor_loads_done();
            const int64_t key = (begin + c) * S::block;
            if (key < all_first || key + S::block > all_end) {
                const int low = (int)min(max(first - key, (int64_t)0), (int64_t)S::block), high = (int)min(max(end - key, (int64_t)0), (int64_t)S::block);
#pragma unroll
                for (int i = 0; i < S::block; ++i) x[i] = i >= low && i < high ? x[i] : masked;
            }
            float best = x[0];
            if (turned) {
#pragma unroll
                for (int i = 1; i < S::block; ++i) best = fminf(best, x[i]);
            } else {
                float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int i = 4; i < S::block; i += 4) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], x[i + k]);
                }
                best = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            }
            // The reference point moves only where the weights would grow beyond 2^8.
            const float grown = top == masked ? (best == masked ? 0.0f : -kNone) : (best - top) * factor;
            const bool moves = grown > kMostGrowth;
            float less = 1.0f;
            if (moves) {
                less = top == masked ? 0.0f : exp2_approx(-grown);
                top = best;
                total *= less;
            }
            if constexpr (S::parts == 3) {
                if (c > 0) {  // the last block's context, relative to the old reference point
                    fine = wait(&context_full[0], (c - 1) & 1);
                    if (!fine) break;
                    tensor_fence_after();
                    add_block();
                }
                if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                    for (int i = 0; i < kSums; ++i) context[i] *= less;
                }
            } else if (c > 0 && __any_sync(0xffffffffu, moves)) {
#pragma unroll 1
                for (int i = 0; i < launch.dims16; i += 32) {
                    float o[32];
                    tensor_load32(context_at + i, o);
                    tensor_loads_done();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] *= less;
                    tensor_store32(context_at + i, reinterpret_cast<const uint32_t*>(o));
                }
            }
            constexpr float lift = __is_same(Elem, __half) ? kHalfLift : 0.0f;
            const float offset = top == masked ? 0.0f : fmaf(-top, factor, lift);
            float2 sums[2] = {both(0.0f), both(0.0f)};
#pragma unroll
            for (int i = 0; i < S::block; i += 32) {
                uint32_t packed[S::parts][16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    float2 w = fma_pair(make_float2(x[i + k], x[i + k + 1]), both(factor), both(offset));
                    w = make_float2(exp2_approx(w.x), exp2_approx(w.y));
                    sums[k / 2 % 2] = add_pair(sums[k / 2 % 2], w);
                    if constexpr (S::parts == 1) packed[0][k / 2] = pack(w.x, w.y, Elem{});
                    else split_weights(w, packed[0][k / 2], packed[1][k / 2], packed[2][k / 2]);
                }
#pragma unroll
                for (int part = 0; part < S::parts; ++part) tensor_store16(lanes + S::weight_at(place, part) + i / 2, packed[part]);
                if (S::parts == 1 && i + 32 == S::block / 2) {
                    tensor_stores_done();
                    tensor_fence_before();
                    barrier_arrive(&weight_full[t][0]);
                }
            }
            total += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
            tensor_stores_done();
            tensor_fence_before();
            barrier_arrive(&weight_full[t][S::parts == 1 ? 1 : 0]);
        }
        if (count > 0 && fine) {
            fine = wait(&context_full[t], S::parts == 1 ? 0 : (count - 1) & 1);
            tensor_fence_after();
        }
        // A sum of 0: the row sees nothing, or (as in any softmax, NaN) scores of -inf alone.
        const auto sum_of = [&](float sum, bool sees) { return sum == 0.0f && sees ? __int_as_float(0x7fffffff) : sum; };
        // Eight dimensions of a row's context, times what makes its weights add up to one.
        const auto put = [&](int64_t to, int of_head, int d, const float* o, float sum) {
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
            Out* out = static_cast<Out*>(p.out) + ((q_begin + to) * p.heads + of_head) * p.head_dim + d;
            if constexpr (sizeof(Out) == 4) {
                float4 a = make_float4(o[0] * inverse, o[1] * inverse, o[2] * inverse, o[3] * inverse);
                float4 c = make_float4(o[4] * inverse, o[5] * inverse, o[6] * inverse, o[7] * inverse);
                if (sum == 0.0f) a = c = make_float4(0, 0, 0, 0);
                reinterpret_cast<float4*>(out)[0] = a;
                reinterpret_cast<float4*>(out)[1] = c;
            } else {
                uint4 a = make_uint4(pack(o[0] * inverse, o[1] * inverse, Elem{}), pack(o[2] * inverse, o[3] * inverse, Elem{}),
                                     pack(o[4] * inverse, o[5] * inverse, Elem{}), pack(o[6] * inverse, o[7] * inverse, Elem{}));
                if (sum == 0.0f) a = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(out) = a;
            }
        };
        if (pieced && pieces > 1 && S::tiles == 2 && fine && counts[1 - t] > 0) fine = wait(&context_full[1 - t], 0, most + 1);  // (shared memory is free then)
        if (fine) {
            float4* fours = reinterpret_cast<float4*>(shared) + t * (S::tile_floats / 4) + (warp % 4) * 32 + lane;
            if (count > 0) add_block();
            const float sum = sum_of(total, end > first);
#pragma unroll
            for (int i = 0; i < S::dims; i += 32) {
                if (i >= p.head_dim) break;
                float o[32];
                if constexpr (S::parts == 3) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = context[i + k];
                } else if (count > 0) {
                    tensor_load32(context_at + i, o);
                    tensor_loads_done();
                }
                if (!pieced || pieces == 1) {
                    if (real) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            if (i + k >= p.head_dim) break;
                            put(row, head, i + k, o + k, sum);
                        }
                    }
                } else if (count > 0) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) fours[(i + k) / 4 * kTileRows] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
            if (pieced && pieces > 1) {
                reinterpret_cast<float2*>(shared)[(t * S::tile_floats + kTileRows * S::dims) / 2 + (warp % 4) * 32 + lane] = make_float2(top, total);
            }
        }
        if (pieced && pieces > 1) {
            // Every CTA joins its share of the rows, out of all pieces' shared memory.  (Every warp comes here, whatever its waits have come to.)
            cluster_meets();
            const int rows = (kRows + pieces - 1) / pieces, parts = (S::tiles * 128) / rows, mine = threadIdx.x % rows, joined = number * rows + mine;
            const int tile = joined / kTileRows, of_tile = joined % kTileRows;
            const int64_t to = row_of(tile, of_tile);
            if (joined < kRows && is_row(of_tile, to) && (int)threadIdx.x / rows < parts) {
                float less[kMostPieces], sum = 0.0f, high = masked;  // what a piece counts for; negative: it has nothing
                float2 ends_at[kMostPieces];
#pragma unroll
                for (int b = 0; b < kMostPieces; ++b) {
                    ends_at[b] = make_float2(masked, 0.0f);
                    if (b < pieces) ends_at[b] = load_of_peer<float2>(q_at + (tile * S::tile_floats + kTileRows * S::dims + 2 * of_tile) * 4, b);
                    high = turned ? fminf(high, ends_at[b].x) : fmaxf(high, ends_at[b].x);
                }
#pragma unroll
                for (int b = 0; b < kMostPieces; ++b) {
                    // (a sum that is NaN counts, so that it is seen)
                    const bool nothing = ends_at[b].x == masked && ends_at[b].y == 0.0f;
                    less[b] = nothing ? -1.0f : ends_at[b].x == high ? 1.0f : exp2_approx((ends_at[b].x - high) * factor);
                    sum += nothing ? 0.0f : less[b] * ends_at[b].y;
                }
                sum = sum_of(sum, sight.end(to) > sight.first(to));
                for (int d = (int)threadIdx.x / rows * 8; d < p.head_dim; d += parts * 8) {
                    float o[8] = {};
#pragma unroll
                    for (int b = 0; b < kMostPieces; ++b) {
                        if (less[b] == -1.0f) continue;
                        const uint32_t from = q_at + (tile * S::tile_floats + (d / 4 * kTileRows + of_tile) * 4) * 4;
                        const float4 x = load_of_peer<float4>(from, b), y = load_of_peer<float4>(from + kTileRows * 16, b);
                        o[0] += x.x * less[b], o[1] += x.y * less[b], o[2] += x.z * less[b], o[3] += x.w * less[b];
                        o[4] += y.x * less[b], o[5] += y.y * less[b], o[6] += y.z * less[b], o[7] += y.w * less[b];
                    }
                    put(to, head0 + of_tile % launch.packed, d, o, sum);
                }
            }
        }
        tensor_fence_before();
    } else {
        few_registers();
    }
    if (pieced && pieces > 1) {
        if (warp >= S::tiles * 4) cluster_meets();
        cluster_meets();  // (its shared memory is read by others until then)
    }
    __syncthreads();
    if (warp == kIssueWarp) {
        tensor_fence_after();
        tensor_free(tensor, 512);
    }
    if (threadIdx.x == 0 && give_up && p.status) atomicOr(p.status, 1);
}

// Keys or values as three bf16 numbers each, (part, position, head, dimension).
__global__ void split_kernel(const float* from, __nv_bfloat16* to, int64_t positions, int64_t stride, int width) {
    const int64_t fours = positions * (width / 4), all = positions * width;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < fours; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t position = i / (width / 4), at = i % (width / 4) * 4;
        const float4 x = __ldg(reinterpret_cast<const float4*>(from + position * stride + at));
        uint2 parts[3];
        split_pair(x.x, x.y, parts[0].x, parts[1].x, parts[2].x);
        split_pair(x.z, x.w, parts[0].y, parts[1].y, parts[2].y);
#pragma unroll
        for (int part = 0; part < 3; ++part) *reinterpret_cast<uint2*>(to + part * all + position * width + at) = parts[part];
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

// (dimension, head, position): boxes of 64 dimensions of `packed` heads and `rows` positions.
bool encode(CUtensorMap* map, bool bfloat, const void* at, int64_t positions, int64_t stride, int heads, int head_dim, int rows, int packed = 1) {
    const cuuint64_t sizes[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)std::max<int64_t>(positions, 1)};
    const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)packed, (cuuint32_t)rows}, steps[3] = {1, 1, 1};
    return encoder()(map, bfloat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(at), sizes, strides, box, steps,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Groups of rows where a tile has `packed` heads: no more than these.
template <class S>
int64_t groups_of_rows(const PromptAttentionParams& p, int packed) {
    return (p.total_q / (S::tiles * (kTileRows / packed)) + p.batch) * (p.heads / packed);
}

// Heads of one kv head that a tile takes together, a divisor of them up to 16: as few as keep the CTAs to one for an SM (they are quicker with
// few rows: one prompt of 100 positions with 8 heads on 2 takes 10.3 us by one head, 12.3 by four), else as many as there are: short
// sequences fill the tiles then (20 of up to 28 positions behind 416, 64 heads on 8, fp32: 78 us instead of 211; five of up to 1501
// with 16 on 4: 214 instead of 230).
template <class S>
int heads_packed(const PromptAttentionParams& p, int sm_count) {
    const int group = p.heads / p.kv_heads;
    int packed = 1;
    for (int d = 1; d <= std::min(group, 16); ++d) {
        if (group % d != 0) continue;
        packed = d;
        if (groups_of_rows<S>(p, d) <= sm_count) break;
    }
    return packed;
}

template <class Elem, class Out, class S>
cudaError_t launch(const PromptAttentionParams& p, int sm_count, cudaStream_t stream, int* launches) {
    constexpr bool bfloat = __is_same(Elem, __nv_bfloat16);
    // Where the groups of rows leave half of the SMs idle, clusters share the keys of each (lengths are not known here: a CTA that finds
    // nothing to do ends early).
    const int packed = heads_packed<S>(p, sm_count), positions = kTileRows / packed;
    const int64_t blocks = groups_of_rows<S>(p, packed);
    const int pieces = (int)std::max<int64_t>(1, std::min({sm_count / blocks, p.total_k / S::block + 1, (int64_t)kMostPieces}));
    static OncePerDevice raised[2];
    const auto kernel = pieces > 1 ? prompt_attention_kernel<Elem, Out, S, true> : prompt_attention_kernel<Elem, Out, S, false>;
    // 1024 bytes to start on a boundary of that.  More than half of an SM's, so that a CTA has the tensor memory for itself.
    const size_t shared = S::shared + 1024 + (size_t)(p.batch + 1) * sizeof(int);
    static_assert(S::shared + 1024 > 114 << 10 && S::shared + 1024 + (kMostPrefixRows + 1) * sizeof(int) <= 227 << 10);
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return e;
    const cudaError_t e = raised[pieces > 1].run(device, [&] {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(S::shared + 1024 + (kMostPrefixRows + 1) * sizeof(int)));
    });
    if (e != cudaSuccess) return e;
    PromptLaunch l;
    l.p = p;
    l.steps = (p.head_dim + 15) / 16;
    l.dims16 = l.steps * 16;
    l.pieces = pieces, l.packed = packed, l.positions = positions;
    const void *k = p.k, *v = p.v;
    int64_t k_rows = p.total_k, k_stride = p.k_stride, v_stride = p.v_stride;
    if constexpr (S::parts == 3) {
        auto* to = static_cast<__nv_bfloat16*>(p.split);
        const auto split = [&](const void* from, int64_t positions, int64_t stride, int heads) {
            const int width = heads * p.head_dim;
            __nv_bfloat16* parts = to;
            to += 3 * positions * width;
            if (positions > 0) {
                const int64_t blocks = (positions * (width / 4) + 255) / 256;
                split_kernel<<<(unsigned)std::min<int64_t>(blocks, (int64_t)sm_count * 8), 256, 0, stream>>>(static_cast<const float*>(from), parts, positions, stride, width);
                ++*launches;
            }
            return parts;
        };
        k = split(p.k, p.total_k, p.k_stride, p.kv_heads);
        v = split(p.v, p.total_k, p.v_stride, p.kv_heads);
        k_rows *= 3;
        k_stride = v_stride = (int64_t)p.kv_heads * p.head_dim;
    }
    if (p.total_k == 0) k = v = p.q, k_stride = v_stride = (int64_t)p.kv_heads * p.head_dim;  // (never read)
    if ((S::parts == 1 && !encode(&l.q_map, bfloat, p.q, p.total_q, p.q_stride, p.heads, p.head_dim, positions, packed)) ||
        !encode(&l.k_map, bfloat, k, k_rows, k_stride, p.kv_heads, p.head_dim, S::block) ||
        !encode(&l.v_map, bfloat, v, k_rows, v_stride, p.kv_heads, p.head_dim, S::block)) {
        return cudaErrorInvalidValue;
    }
    if (pieces > 1) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(blocks * pieces));
        config.blockDim = dim3(S::threads);
        config.dynamicSmemBytes = shared;
        config.stream = stream;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = (unsigned)pieces, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = 1;
        if (const cudaError_t failed = cudaLaunchKernelEx(&config, kernel, l)) return failed;
    } else {
        kernel<<<(unsigned)blocks, S::threads, shared, stream>>>(l);
    }
    ++*launches;
    return cudaGetLastError();
}

template <class Elem, class Out, int parts>
cudaError_t launch_dims(const PromptAttentionParams& p, int sm_count, cudaStream_t stream, int* launches) {
    if (p.head_dim <= 64) return launch<Elem, Out, Shape<64, parts>>(p, sm_count, stream, launches);
    return launch<Elem, Out, Shape<128, parts>>(p, sm_count, stream, launches);
}

}  // namespace

size_t prompt_split_bytes(const PromptAttentionParams& p) {
    if (p.type != kFloat32) return 0;
    return (size_t)12 * p.head_dim * p.total_k * p.kv_heads;
}

cudaError_t launch_prompt_attention(const PromptAttentionParams& p, int sm_count, cudaStream_t stream, int* launches) {
    *launches = 0;
    if (!encoder()) return cudaErrorNotSupported;
    if (p.type == kFloat32) return launch_dims<__nv_bfloat16, float, 3>(p, sm_count, stream, launches);
    if (p.type == kBfloat16) return launch_dims<__nv_bfloat16, __nv_bfloat16, 1>(p, sm_count, stream, launches);
    return launch_dims<__half, __half, 1>(p, sm_count, stream, launches);
}

}  // namespace psx
