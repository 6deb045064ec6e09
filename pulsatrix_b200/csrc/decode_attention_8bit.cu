// Attention of the new positions over a cache held in 8 bits, in one pass over the cache.
//
// For a query row q and cached position j with codes k_j, v_j and block scales a_j, b_j:
//     s_j = scale * a_j * (q . k_j),   context = sum_j exp(s_j) b_j v_j / sum_j exp(s_j)   over the positions that the row sees.
//
// Codes become halves exactly, so both products run as half matrix instructions (m16n8k16, float accumulators) in the
// transposed form: 16 positions by 8 query rows, then 16 dimensions by 8 query rows.  The query rows of a kv head (group x
// new positions, up to 16) are the narrow side, which wastes nothing at 8 rows; the codes are converted once for all of them.
// A query row is brought to between 2^14 and 2^15 and rounded to halves (bf16 and fp16 queries lose nothing but bits below 2^-38 of
// their largest element); an fp32 row is a half and the half that is left, two instructions each: 22 bits for elements down to 2^-17 of
// the largest, for those below 2^-39 of that.  Weights:
// the running maximum M is taken over s_j + log2(b_j) - 15, so that w_j = exp(s_j - M) b_j is at most 2^15 whatever the scales; it is
// rounded to halves (2^-11, below the rounding of a bf16 or fp16 context; for fp32 contexts again two halves).  Halves reach from
// 65,504 down to 2^-14 with all their bits and end at 2^-24, so a weight has its 11 bits down to 2^-29 of the largest, and the 22 of two down
// to 2^-18 (brought to 1 instead, weights below 2^-25 of the largest were lost: many of them behind one that leads by 18 nats
// are all of a context whose first value is 0).  Maxima, sums and contexts are floats.
//
// A (row, kv head) pair's cached positions are cut into tiles of 32, and the tiles into pieces, a block each: as many as fill the GPU
// once, or as pieces of 128 tiles make where that is more, which evens out rows of different lengths (64 rows x 8 kv heads of up to 8191
// positions, in a graph: 167 us as one piece each, 141 to 145 as two from box to box; pieces of 64 tiles: 138, but 96 rows x 1 of up to
// 16,000: 70 instead of 61.  A call among others, with a cold L2: 157).  The last block of a pair to end joins its pieces, in order.
// (Equal shares of all pairs' tiles laid on one axis: 139 us there,
// with a cold L2 143 instead of 155; but 64 x 8 of 1000: 41 instead of 25, 24 x 8 of up to 4096: 52 instead of 33, since most blocks then have
// the end of one pair and the start of another.)  Inside a block each of four warps takes every fourth tile, with
// its own two stages of 32 positions in shared memory (cp.async, 16 bytes a lane), so that no warp waits for another until the end.
// Bound by HBM for long caches (2 bytes per position, head dimension and kv head), by the chain of a tile for short ones: some 2100
// clocks from a tile's arrival to its weights' products, most of them conversions of codes (64 instructions for 32 positions x 64
// dimensions, two clocks each).
#include "decode_attention_8bit.cuh"

#include <algorithm>

#include "elements.cuh"
#include "once_per_device.hpp"

namespace psx {
namespace {

constexpr int kThreads = 128, kWarps = 4, kTile = 32;
constexpr int kStages = 2;       // of a warp: the tile in work and the one on its way
constexpr int kMostShare = 128;  // tiles that a block takes where shorter pieces only balance
constexpr float kNone = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kQueryLift = 14;        // a query row's largest element has the exponent 14: halves end at 65,504
constexpr float kWeightLift = 15.0f;  // the largest weight is 2^15
// The least value scale for which that holds; below it weights are smaller, by its ratio to this.  A weight without its scale is 2^97 at most
// then, and 2^30 of them (the longest cache) add up to a float.
constexpr float kLeastScale = 0x1p-82f;

__host__ __device__ constexpr int stage_bytes(int dims) { return 2 * kTile * dims + 16; }  // keys, values, two scales each
__host__ __device__ constexpr size_t shared_of(int dims) { return (size_t)kWarps * kStages * stage_bytes(dims); }

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void multiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t halves(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    uint32_t r;
    __builtin_memcpy(&r, &h, 4);
    return r;
}
// What the halves leave of the two floats, as halves.
__device__ __forceinline__ uint32_t halves_left(float low, float high, uint32_t taken) {
    __half2 h;
    __builtin_memcpy(&h, &taken, 4);
    const float2 t = __half22float2(h);
    return halves(low - t.x, high - t.y);
}

template <class T>
__device__ __forceinline__ void store_four(T* to, float4 x, float factor) {
    alignas(16) const T four[4] = {from_float<T>(x.x * factor), from_float<T>(x.y * factor), from_float<T>(x.z * factor), from_float<T>(x.w * factor)};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(four);
    else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(four);
}

// Chunk (16 codes) `chunk` of row `row` of a stage lies at this chunk of the row: eight rows' chunks of one column lie in
// different banks, and so do four neighbouring chunks of two neighbouring rows.
template <int dims>
__device__ __forceinline__ int placed(int row, int chunk) {
    if constexpr (dims == 64) return chunk ^ ((row >> 1) & 3);
    else return chunk ^ (((row & 1) << 2) | ((row >> 1) & 3));
}

// Bounds of what query rows see, in positions.
struct Sight {
    int length, first_own;  // the position of the first new one
    int window;             // 0: none
    __device__ __forceinline__ int last(int i, bool causal) const { return causal ? first_own + i : length - 1; }
    __device__ __forceinline__ int first(int i) const { return window > 0 ? first_own + i - window + 1 : 0; }
    __device__ __forceinline__ int first_tile() const { return max(first(0), 0) / kTile; }
    __device__ __forceinline__ int end_tile() const { return (length + kTile - 1) / kTile; }
};

__device__ __forceinline__ Sight sight_of(const Attention8bitParams& p, int row) {
    const int length = (int)min(max(p.lengths[row], (int64_t)0), p.cache.max_len);
    return {length, length - p.q_len, p.causal ? (int)p.window : 0};
}

template <class T, int dims, int tiles_of_rows>
__global__ void __launch_bounds__(kThreads, dims == 256 ? 1 : tiles_of_rows == 2 && dims == 128 ? 2 : dims == 128 ? 3 : 4) decode_attention_8bit_kernel(const __grid_constant__ Attention8bitParams p) {
    constexpr bool precise = sizeof(T) == 4;
    constexpr int kStageBytes = stage_bytes(dims), kSegments = dims / 64, kBlocks = dims / 16;
    constexpr int kRows = 8 * tiles_of_rows;
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ float tops[kWarps][kRows], totals[kWarps][kRows];
    __shared__ int is_last;
    const Cache8bitView& c = p.cache;
    const int head_dim = c.head_dim, chunks = head_dim / 16;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, gid = lane / 4, tig = lane % 4;
    uint8_t* stages = shared + warp * kStages * kStageBytes;
    const uint32_t stages_at = shared_address(stages);
    const int shift = 31 - __clz(c.block);

    // This block's pair (its query rows from first_row on, eight at a time beyond 128 dimensions), and its tiles of the pair's.
    const int64_t unit = blockIdx.x / (unsigned)p.pieces, pair = dims == 256 ? unit / p.row_groups : unit;
    const int first_row = dims == 256 ? (int)(unit % p.row_groups) * kRows : 0, rows = dims == 256 ? min(p.rows - first_row, kRows) : p.rows;
    const int number = (int)(blockIdx.x % (unsigned)p.pieces), row = (int)(pair / c.kv_heads), head = (int)(pair % c.kv_heads);
    const Sight sight = sight_of(p, row);
    const int tiles = max(sight.end_tile() - sight.first_tile(), 0);
    const int share = max(max(kWarps, (tiles + p.pieces - 1) / p.pieces), min((tiles + p.spread - 1) / p.spread, kMostShare));
    const int from_tile = number * share, to_tile = min(tiles, from_tile + share);
    const int64_t first_element = (((int64_t)row * p.heads + (int64_t)head * p.group) * p.q_len + first_row) * head_dim;
    T* context = static_cast<T*>(p.context) + first_element;
    if (from_tile >= to_tile) {
        if (tiles == 0 && number == 0) {  // a row that sees nothing
            for (int i = threadIdx.x; i < rows * head_dim; i += kThreads) context[i] = from_float<T>(0.0f);
        }
        return;
    }
    const int tile0 = sight.first_tile();
    const uint8_t* keys = c.key_codes + pair * c.max_len * head_dim;
    const uint8_t* values = c.value_codes + pair * c.max_len * head_dim;
    const float* key_scales = c.key_scales + pair * c.blocks;
    const float* value_scales = c.value_scales + pair * c.blocks;

    const int seen = max(sight.first(0), 0);  // no row sees a position before this one
    const auto fetch = [&](int tile, int stage) {  // positions that no row sees arrive as zeros, whatever the cache holds there
        const int position = (tile0 + tile) * kTile;
        const uint32_t to = stages_at + stage * kStageBytes;
        if (head_dim == dims && position >= seen && position + kTile <= sight.length) {  // 32 whole rows, one run of memory
            const uint8_t* from = keys + (int64_t)position * dims + lane * 16;
            const int64_t apart = values - keys;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                const int r = (i * 32 + lane) / kBlocks, chunk = lane % kBlocks;
                const uint32_t place = to + r * dims + placed<dims>(r, chunk) * 16;
                copy16(place, from + i * 512);
                copy16(place + kTile * dims, from + apart + i * 512);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < kBlocks; ++i) {
                const int index = i * 32 + lane, r = index / kBlocks, chunk = index % kBlocks;
                if (chunk < chunks) {
                    const bool there = position + r < sight.length && position + r >= seen;
                    const int64_t offset = there ? (int64_t)(position + r) * head_dim + chunk * 16 : 0;
                    const uint32_t place = to + r * dims + placed<dims>(r, chunk) * 16;
                    copy16(place, keys + offset, there);
                    copy16(place + kTile * dims, values + offset, there);
                }
            }
        }
        if (lane < 4) {  // the scales of the tile's two halves, keys' then values' (of a half that no row sees, 0 too: a NaN times 0 is one)
            const int first = position + lane % 2 * 16;
            const bool there = first < sight.length && first + 16 > seen;
            copy4(to + 2 * kTile * dims + lane * 4, (lane < 2 ? key_scales : value_scales) + (there ? first >> shift : 0), there);
        }
    };
    if (from_tile + warp < to_tile) fetch(from_tile + warp, 0);

    // The query rows as the right-hand operand: lane (gid, tig) holds row gid's dimensions 16 tig .. 16 tig + 15 of every 64.
    uint32_t qh[tiles_of_rows][kSegments][4][2], ql[precise ? tiles_of_rows : 1][precise ? kSegments : 1][4][2];
    float row_scale[tiles_of_rows][2];  // of the score rows that this lane holds: rows 2 tig and 2 tig + 1
    const T* q = static_cast<const T*>(p.q) + first_element;
#pragma unroll
    for (int n = 0; n < tiles_of_rows; ++n) {
        const int r = n * 8 + gid;
        float x[kSegments][16];
        float largest = 0.0f;
#pragma unroll
        for (int s = 0; s < kSegments; ++s) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = s * 64 + tig * 16 + i;
                float4 four = make_float4(0, 0, 0, 0);
                if (r < rows && d < head_dim) four = load_four(q + (int64_t)r * head_dim + d);
                x[s][i] = four.x, x[s][i + 1] = four.y, x[s][i + 2] = four.z, x[s][i + 3] = four.w;
                largest = fmaxf(largest, fmaxf(fmaxf(fabsf(four.x), fabsf(four.y)), fmaxf(fabsf(four.z), fabsf(four.w))));
            }
        }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^-e with largest = m 2^(14 + e), 1 <= m < 2, for every finite row (of tiny ones no more than 2^114: both powers are normal numbers)
        const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -100), 127) - kQueryLift;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int s = 0; s < kSegments; ++s) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float low = x[s][4 * w + 2 * h] * down, high = x[s][4 * w + 2 * h + 1] * down;
                    qh[n][s][w][h] = halves(low, high);
                    if constexpr (precise) ql[n][s][w][h] = halves_left(low, high, qh[n][s][w][h]);
                }
            }
        }
        const float factor = up * (p.scale * kLog2e);
        row_scale[n][0] = __shfl_sync(0xffffffffu, factor, 8 * tig);      // (row 2 tig is lanes 8 tig .. 8 tig + 3)
        row_scale[n][1] = __shfl_sync(0xffffffffu, factor, 8 * tig + 4);
    }

    float out[tiles_of_rows][kBlocks][4], top[tiles_of_rows][2], total[tiles_of_rows][2];
#pragma unroll
    for (int n = 0; n < tiles_of_rows; ++n) {
        top[n][0] = top[n][1] = kNone;
        total[n][0] = total[n][1] = 0.0f;
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) out[n][m][0] = out[n][m][1] = out[n][m][2] = out[n][m][3] = 0.0f;
    }
    // Positions that every row sees need no mask.
    const int all_from = sight.first(p.q_len - 1), all_to = sight.last(0, p.causal != 0);

    int stage = 0;
    for (int tile = from_tile + warp; tile < to_tile; tile += kWarps) {
        copies_done();
        __syncwarp();
        if (tile + kWarps < to_tile) fetch(tile + kWarps, stage ^ 1);  // (where the tile before this one was)
        const uint8_t* k_stage = stages + stage * kStageBytes;
        const float* scales = reinterpret_cast<const float*>(k_stage + 2 * kTile * dims);
        const int position = (tile0 + tile) * kTile;
        float score[tiles_of_rows][2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int n = 0; n < tiles_of_rows; ++n) score[n][half][0] = score[n][half][1] = score[n][half][2] = score[n][half][3] = 0.0f;
            const int r0 = half * 16 + gid, r1 = r0 + 8;
#pragma unroll
            for (int s = 0; s < kSegments; ++s) {
                const int chunk = s * 4 + tig;
                uint4 a = make_uint4(0, 0, 0, 0), b = a;
                if (chunk < chunks) {
                    a = *reinterpret_cast<const uint4*>(k_stage + r0 * dims + placed<dims>(r0, chunk) * 16);
                    b = *reinterpret_cast<const uint4*>(k_stage + r1 * dims + placed<dims>(r1, chunk) * 16);
                }
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_halves(aw[w], a0, a2);
                    codes_to_halves(bw[w], a1, a3);
#pragma unroll
                    for (int n = 0; n < tiles_of_rows; ++n) {
                        if constexpr (precise) multiply(score[n][half], a0, a1, a2, a3, ql[n][s][w][0], ql[n][s][w][1]);
                        multiply(score[n][half], a0, a1, a2, a3, qh[n][s][w][0], qh[n][s][w][1]);
                    }
                }
            }
        }
        // score[n][half][2 o + i]: position half * 16 + 8 o + gid, query row 8 n + 2 tig + i
        float value_scale[2], value_log[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float key_scale = scales[half];
            value_scale[half] = scales[2 + half];
            value_log[half] = __log2f(fmaxf(value_scale[half], kLeastScale)) - kWeightLift;
#pragma unroll
            for (int n = 0; n < tiles_of_rows; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) score[n][half][i] *= key_scale * row_scale[n][i & 1];
            }
        }
        if (position < all_from || position + kTile - 1 > all_to) {
#pragma unroll
            for (int n = 0; n < tiles_of_rows; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int own = (first_row + n * 8 + 2 * tig + i) % p.q_len;
                    const int first = sight.first(own), last = sight.last(own, p.causal != 0);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const int j = position + half * 16 + o * 8 + gid;
                            if (j < first || j > last) score[n][half][2 * o + i] = kNone;
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < tiles_of_rows; ++n) {
            float high[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                high[i] = fmaxf(fmaxf(score[n][0][i], score[n][0][2 + i]) + value_log[0], fmaxf(score[n][1][i], score[n][1][2 + i]) + value_log[1]);
#pragma unroll
                for (int step = 4; step < 32; step *= 2) high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], step));
            }
            if (__any_sync(0xffffffffu, high[0] > top[n][0] || high[1] > top[n][1])) {
                float less[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float next = fmaxf(top[n][i], high[i]);
                    less[i] = next > kNone ? exp2_approx(top[n][i] - next) : 1.0f;
                    top[n][i] = next;
                    total[n][i] *= less[i];
                }
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    out[n][m][0] *= less[0], out[n][m][1] *= less[1];
                    out[n][m][2] *= less[0], out[n][m][3] *= less[1];
                }
            }
        }
        // Weights, rounded to halves and turned round: lane (gid, tig) then holds query row gid's weights of positions 2 tig, 2 tig + 1.
        uint32_t wh[tiles_of_rows][2][2], wl[precise ? tiles_of_rows : 1][2][2];
#pragma unroll
        for (int n = 0; n < tiles_of_rows; ++n) {
            const float t0 = top[n][0] > kNone ? top[n][0] : 0.0f, t1 = top[n][1] > kNone ? top[n][1] : 0.0f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const float e0 = exp2_approx(score[n][half][2 * o] - t0), e1 = exp2_approx(score[n][half][2 * o + 1] - t1);
                    total[n][0] += e0;
                    total[n][1] += e1;
                    const float w0 = e0 * value_scale[half], w1 = e1 * value_scale[half];
                    const uint32_t taken = halves(w0, w1);
                    wh[n][half][o] = transposed(taken);
                    if constexpr (precise) wl[n][half][o] = transposed(halves_left(w0, w1, taken));
                }
            }
        }
        // The values come as 8 x 8 matrices of code pairs, turned round: lane (gid, tig) gets dimensions 2 gid, 2 gid + 1 of
        // positions 2 tig and 2 tig + 1; dimension 2 gid is row gid of the left-hand operand, 2 gid + 1 row gid + 8.
        const uint32_t v_at = stages_at + stage * kStageBytes + kTile * dims;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = half * 16 + lane % 16;
#pragma unroll
            for (int m = 0; m < kBlocks; m += 2) {
                if (m < chunks) {
                    uint32_t x[4];
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                        : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                        : "r"(v_at + r * dims + placed<dims>(r, m + lane / 16) * 16)
                        : "memory");
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t low = __byte_perm(x[2 * i], 0, 0x3120), high = __byte_perm(x[2 * i + 1], 0, 0x3120);
                        uint32_t a0, a1, a2, a3;
                        codes_to_halves(low, a0, a1);
                        codes_to_halves(high, a2, a3);
#pragma unroll
                        for (int n = 0; n < tiles_of_rows; ++n) {
                            if constexpr (precise) multiply(out[n][m + i], a0, a1, a2, a3, wl[n][half][0], wl[n][half][1]);
                            multiply(out[n][m + i], a0, a1, a2, a3, wh[n][half][0], wh[n][half][1]);
                        }
                    }
                }
            }
        }
        stage ^= 1;
    }

    // The four warps' results meet in shared memory.  (The stages are free: every warp has read its own.)
#pragma unroll
    for (int n = 0; n < tiles_of_rows; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int step = 4; step < 32; step *= 2) total[n][i] += __shfl_xor_sync(0xffffffffu, total[n][i], step);
            if (gid == 0) {
                tops[warp][n * 8 + 2 * tig + i] = top[n][i];
                totals[warp][n * 8 + 2 * tig + i] = total[n][i];
            }
        }
    }
    __syncthreads();
    float* meet = reinterpret_cast<float*>(shared);  // (warp, row, dimension)
#pragma unroll
    for (int n = 0; n < tiles_of_rows; ++n) {
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = n * 8 + 2 * tig + (i & 1), d = m * 16 + 2 * gid + (i >> 1);
                meet[(warp * kRows + r) * dims + d] = out[n][m][i];
            }
        }
    }
    __syncthreads();
    // What makes a row's weights add up to one.  A sum of 0: the row sees nothing, or (as in any softmax, NaN) scores of -inf alone.
    const auto inverse_of = [&](int r, float sum) {
        if (sum != 0.0f) return 1.0f / sum;
        const int own = (first_row + r) % p.q_len;
        return sight.last(own, p.causal != 0) < max(sight.first(own), 0) ? 0.0f : __int_as_float(0x7fffffff);
    };
    const bool whole = from_tile == 0 && to_tile == tiles;
    const int piece_floats = kRows * (dims + 4);  // (a row's context, its maximum and sum, two unused)
    const int fours = head_dim / 4;
    float* piece = p.partial + (int64_t)blockIdx.x * piece_floats;
    for (int i = threadIdx.x; i < rows * fours; i += kThreads) {
        const int r = i / fours, d = i % fours * 4;
        float high = kNone, sum = 0.0f;
        float4 value = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) high = fmaxf(high, tops[w][r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (totals[w][r] == 0.0f) continue;  // (a warp without a position that the row sees)
            const float less = exp2_approx(tops[w][r] - high);
            const float4 part = *reinterpret_cast<const float4*>(meet + (w * kRows + r) * dims + d);
            sum += totals[w][r] * less;
            value.x += part.x * less, value.y += part.y * less, value.z += part.z * less, value.w += part.w * less;
        }
        if (whole) {
            store_four(context + r * head_dim + d, value, inverse_of(r, sum));
        } else {
            __stcg(reinterpret_cast<float4*>(piece + r * (dims + 4) + d), value);
            if (d == 0) __stcg(reinterpret_cast<float2*>(piece + r * (dims + 4) + dims), make_float2(high, sum));
        }
    }
    if (!whole) {
        const int pieces = (tiles + share - 1) / share;
        __syncthreads();
        if (threadIdx.x == 0) {  // (release: the block's pieces, ordered before by the barrier; acquire: the other blocks')
            int before;
            asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + unit) : "memory");
            is_last = before == pieces - 1;
            if (is_last) p.arrived[unit] = 0;
        }
        __syncthreads();
        if (is_last) {
            const auto piece_of = [&](int b) { return p.partial + (unit * p.pieces + b) * piece_floats; };
            // A thread's part of the first pieces' contexts is asked for along with their maxima and sums.
            constexpr int kAhead = 8;
            const int mine_row = threadIdx.x / fours, mine_d = threadIdx.x % fours * 4;
            const bool mine_real = mine_row < rows;
            float4 ahead[kAhead];
#pragma unroll
            for (int b = 0; b < kAhead; ++b) {
                ahead[b] = make_float4(0, 0, 0, 0);
                if (b < pieces && mine_real) ahead[b] = __ldcg(reinterpret_cast<const float4*>(piece_of(b) + mine_row * (dims + 4) + mine_d));
            }
            float2* less = reinterpret_cast<float2*>(shared);  // (piece, row): maximum and sum, then what the piece counts for
            for (int i = threadIdx.x; i < pieces * rows; i += kThreads) {
                less[i] = __ldcg(reinterpret_cast<const float2*>(piece_of(i / rows) + i % rows * (dims + 4) + dims));
            }
            __syncthreads();
            for (int r = warp; r < rows; r += kWarps) {
                float high = kNone, sum = 0.0f;
                for (int b = lane; b < pieces; b += 32) high = fmaxf(high, less[b * rows + r].x);
#pragma unroll
                for (int step = 16; step > 0; step /= 2) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, step));
                for (int b = lane; b < pieces; b += 32) {
                    const float2 mine = less[b * rows + r];
                    const float factor = mine.x > kNone ? exp2_approx(mine.x - high) : 0.0f;
                    less[b * rows + r].x = factor;
                    sum += factor * mine.y;
                }
#pragma unroll
                for (int step = 16; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
                if (lane == 0) totals[0][r] = sum;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < rows * fours; i += kThreads) {
                const int r = i / fours, d = i % fours * 4;
                float4 value = make_float4(0, 0, 0, 0);
                const auto add = [&](const float4& part, float factor) {
                    value.x += part.x * factor, value.y += part.y * factor, value.z += part.z * factor, value.w += part.w * factor;
                };
                int b = 0;
                if (i == threadIdx.x) {
#pragma unroll
                    for (; b < kAhead; ++b) {
                        if (b < pieces) add(ahead[b], less[b * rows + r].x);
                    }
                }
#pragma unroll 8
                for (; b < pieces; ++b) add(__ldcg(reinterpret_cast<const float4*>(piece_of(b) + r * (dims + 4) + d)), less[b * rows + r].x);
                store_four(context + r * head_dim + d, value, inverse_of(r, totals[0][r]));
            }
        }
    }
}

template <class T, int dims, int tiles_of_rows>
cudaError_t launch(const Attention8bitParams& p, cudaStream_t stream) {
    static OncePerDevice raised;
    const auto kernel = decode_attention_8bit_kernel<T, dims, tiles_of_rows>;
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return e;
    const cudaError_t e = raised.run(device, [&] {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_of(dims));
    });
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)(p.cache.batch * p.cache.kv_heads * p.row_groups * p.pieces), kThreads, shared_of(dims), stream>>>(p);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_type(const Attention8bitParams& p, cudaStream_t stream) {
    const int dims = p.cache.head_dim;
    if (dims > 128) return launch<T, 256, 1>(p, stream);
    if (dims > 64) return p.rows <= 8 ? launch<T, 128, 1>(p, stream) : launch<T, 128, 2>(p, stream);
    return p.rows <= 8 ? launch<T, 64, 1>(p, stream) : launch<T, 64, 2>(p, stream);
}

int padded_dims(const Attention8bitParams& p) { return p.cache.head_dim > 128 ? 256 : p.cache.head_dim > 64 ? 128 : 64; }

// Query rows of a block's kernel.
int rows_of_block(const Attention8bitParams& p) { return p.rows <= 8 || padded_dims(p) == 256 ? 8 : 16; }

}  // namespace

void plan_attention_8bit(Attention8bitParams& p, int sm_count) {
    const int dims = padded_dims(p);
    p.row_groups = dims == 256 ? (p.rows + 7) / 8 : 1;  // (more rows' contexts do not fit the registers; the cache comes out of L2 the second time)
    const int64_t tiles = (p.cache.max_len + kTile - 1) / kTile, units = p.cache.batch * p.cache.kv_heads * p.row_groups;
    // Blocks that the GPU holds at once, by registers and shared memory.
    const int64_t blocks = (int64_t)sm_count * (dims == 256 ? 1 : dims == 64 ? 4 : p.rows > 8 ? 2 : 3);
    // The pieces of a pair have their maxima and sums in shared memory when they are joined.
    const int64_t most = std::min<int64_t>((tiles + kWarps - 1) / kWarps, shared_of(dims) / (rows_of_block(p) * sizeof(float2)));
    const int64_t spread = std::max<int64_t>(1, blocks / units);
    const int64_t balanced = std::min((tiles + kMostShare - 1) / kMostShare, 8 * blocks / units);  // (blocks that find nothing to do cost time too)
    p.spread = (int)std::min(spread, most);
    p.pieces = (int)std::min(std::max(spread, balanced), most);
}

int64_t attention_8bit_counters(const Attention8bitParams& p) { return p.cache.batch * p.cache.kv_heads * p.row_groups; }

size_t attention_8bit_partial_bytes(const Attention8bitParams& p) {
    return (size_t)(attention_8bit_counters(p) * p.pieces) * rows_of_block(p) * (padded_dims(p) + 4) * sizeof(float);
}

cudaError_t launch_decode_attention_8bit(const Attention8bitParams& p, cudaStream_t stream) {
    if (p.rows > 16 || p.cache.head_dim > 256) return cudaErrorInvalidValue;
    if (p.type == kFloat32) return launch_type<float>(p, stream);
    if (p.type == kBfloat16) return launch_type<__nv_bfloat16>(p, stream);
    return launch_type<__half>(p, stream);
}

}  // namespace psx
