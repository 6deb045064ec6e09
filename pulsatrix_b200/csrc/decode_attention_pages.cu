// Attention of the new positions over a cache in pages, in one pass over the pages that a row uses.
//
//     s_j = scale * (q . k_j),   context = sum_j exp(s_j) v_j / sum_j exp(s_j)   over the positions that the row sees.
//
// Both products run as matrix instructions with float accumulators in the transposed form: 16 positions by 8 query rows (the rows of a
// kv head: group x new positions, up to 16), then 16 dimensions by 8 query rows.  Nothing is staged: a lane loads 16 bytes of a key's row, and
// which dimensions a product's step takes is ours to choose, as long as both sides choose the same; so the loaded words are the
// left-hand operand as they are.  Of the values a lane loads 16 bytes of four positions, and pairs of positions of one dimension
// are put together by byte permutations.  Tiles are 16 positions, so that every tile lies in one page, whatever the page's size.
//   bf16, fp16  one instruction (m16n8k16) per 16 dimensions; weights are a number of the type and what is left of it, two
//               instructions, so that they carry 16 or 22 bits and the context's own rounding is all that is seen.  fp16 weights are 2^15 at most
//               instead of 1 (they end at 2^-24).
//   fp32        every factor as two numbers of 11 bits (tf32), three instructions (m16n8k8): products are exact to about 2^-22.  Sums of several
//               instructions are added up outside of them (inside, the context of 2000 positions was off by 1.3e-6 instead of 2.8e-7).
//
// A (row, kv head) pair's tiles are cut into pieces, a block each, and every warp of a block takes every fourth tile, with the next one's keys on their way
// while this one's values are in work (without: 283 us instead of 257 for 64 rows x 8 kv heads of up to 8191 positions of 128); the last block of
// a pair to end joins the pieces, in order.  (Pieces as the CTAs of a cluster, joined over its shared memory: 12 x 16 fp32 pairs of up to 1999 positions 42 us
// instead of 37, 13 x 4 of up to 5997 47 instead of 34.  Pieces of equal length over all rows, which every block works out from the lengths: 39 and 35.)
// Bound by HBM, the keys and values that are seen, once: that call reads at 6.3 TB/s when it is replayed on the same inputs (258 us; a plain copy runs at 6.5), and at 5.9 to 6.3
// on other inputs every time (260 to 275 us, by the machine); short caches by the chain from a row's length over its pages to the join, some 9 us.
#include "decode_attention_pages.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elements.cuh"
#include "psx_device.cuh"

namespace psx {
namespace {

constexpr int kThreads = 128, kWarps = 4, kTile = 16;
constexpr double kSplitRate = 4.0;  // pieces squared for a tile where few pairs are cut to fill the GPU: more are longer in joining than they save
// Tiles that a block takes where shorter pieces only balance.
__host__ __device__ constexpr int most_share(int dims) { return dims == 256 ? 32 : 64; }
constexpr float kNone = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

template <class T>
struct Kind {
    static constexpr bool precise = sizeof(T) == 4;
    static constexpr int elements = 16 / sizeof(T);          // of 16 bytes
    static constexpr int tiles = precise ? 2 : 4;            // of 16 dimensions that eight lanes' 16 bytes make
    static constexpr float lift = std::is_same<T, __half>::value ? 15.0f : 0.0f;  // the largest weight is 2^lift
};

__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The nearest number of 11 bits, and what is left: 12 bits, of which the instruction takes 11.
__device__ __forceinline__ uint32_t eleven_bits(uint32_t x) { return (x + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t left_of(uint32_t x, uint32_t taken) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(taken)); }

// c += a b with a's four and b's two numbers in two parts each.
__device__ __forceinline__ void multiply_parts(float (&c)[4], const uint32_t (&a)[4], const uint4& b) {
    uint32_t high[4], low[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) high[i] = eleven_bits(a[i]), low[i] = left_of(a[i], high[i]);
    multiply(c, low, b.x, b.y, 0.0f);
    multiply(c, high, b.z, b.w, 0.0f);
    multiply(c, high, b.x, b.y, 0.0f);
}

// Sums of many instructions are added up outside of them: they cut off what does not fit their sum, always toward zero.
__device__ __forceinline__ void add_to(float (&c)[4], const float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] += x[i];
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

template <class T>
__device__ __forceinline__ uint32_t pair_of(float low, float high) {
    const T two[2] = {from_float<T>(low), from_float<T>(high)};
    uint32_t r;
    __builtin_memcpy(&r, two, 4);
    return r;
}
template <class T>
__device__ __forceinline__ uint32_t pair_left(float low, float high, uint32_t taken) {
    T two[2];
    __builtin_memcpy(two, &taken, 4);
    return pair_of<T>(low - to_float(two[0]), high - to_float(two[1]));
}

template <class T>
__device__ __forceinline__ void store_four(T* to, float4 x, float factor) {
    alignas(16) const T four[4] = {from_float<T>(x.x * factor), from_float<T>(x.y * factor), from_float<T>(x.z * factor), from_float<T>(x.w * factor)};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(four);
    else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(four);
}

// Cached positions are read once.  (Coherent, as all loads here: the kernel begins while the one that wrote them may be at its end.)
__device__ __forceinline__ uint4 load_once(const void* at) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(at));
    return r;
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

__host__ __device__ constexpr int words_of(int dims, int bytes) { return dims * bytes / 8; }  // of a tile's keys, a lane's

// Blocks that an SM holds, by registers.
__host__ __device__ constexpr int blocks_of(int dims, int bytes, int tiles_of_rows) {
    if (dims == 256 || (tiles_of_rows == 2 && bytes == 4)) return 2;
    return dims == 128 || tiles_of_rows == 2 ? 3 : 4;
}

// Query rows in shared memory, then the warps' contexts.
__host__ __device__ constexpr size_t shared_of(int dims, int tiles_of_rows, bool precise) {
    const size_t meet = (size_t)kWarps * 8 * tiles_of_rows * dims * sizeof(float), parts = (size_t)tiles_of_rows * dims / (precise ? 8 : 16) * 32 * (precise ? sizeof(uint4) : sizeof(uint2));
    return meet > parts ? meet : parts;
}

template <class T, int dims, int tiles_of_rows>
__global__ void __launch_bounds__(kThreads, blocks_of(dims, sizeof(T), tiles_of_rows))
    decode_attention_pages_kernel(const __grid_constant__ PagedAttentionParams p) {
    using K = Kind<T>;
    constexpr bool precise = K::precise;
    constexpr int E = K::elements, kSteps = dims / (4 * E);  // 16 bytes of a lane for every so many dimensions of a key
    constexpr int kBlocks = dims / 16, kRows = 8 * tiles_of_rows;
    constexpr int kSegment = kSteps < 64 / 8 ? kSteps : 64 / 8;  // of steps whose two rows a lane holds at once
    constexpr bool keys_ahead = words_of(dims, sizeof(T)) <= 32;      // the next tile's keys are on their way while this one's values are in work
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ float tops[kWarps][kRows], totals[kWarps][kRows];
    __shared__ int is_last;
    const PageTableView& t = p.cache.table;
    const int head_dim = p.cache.head_dim, kv_heads = p.cache.kv_heads;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, gid = lane / 4, tig = lane % 4;

    grid_dependency_wait();
    grid_dependents_may_launch();
    // This block's pair (beyond 128 dimensions eight of its query rows), and its tiles of the pair's.
    const int unit = (int)(blockIdx.x / (unsigned)p.pieces), number = (int)(blockIdx.x % (unsigned)p.pieces);
    const int pair = dims == 256 ? unit / p.row_groups : unit, first_row = dims == 256 ? unit % p.row_groups * kRows : 0;
    const int row = pair / kv_heads, head = pair % kv_heads, rows = dims == 256 ? min(p.rows - first_row, kRows) : p.rows;
    const int length = t.length(row);
    const Sight sight{length, length - p.q_len, p.causal ? (int)p.window : 0};
    const int tile0 = sight.first_tile(), tiles = max(sight.end_tile() - tile0, 0);
    const int share = max(max(kWarps, (tiles + p.pieces - 1) / p.pieces), min((tiles + p.spread - 1) / p.spread, most_share(dims)));
    const int from_tile = number * share, to_tile = min(tiles, from_tile + share);
    // Row r of the pair is new position r / group, head r % group of the kv head's.
    const auto element_of = [&](int r) {
        r += first_row;
        return (((int64_t)row * p.q_len + r / p.group) * p.heads + (int64_t)head * p.group + r % p.group) * head_dim;
    };
    T* context = static_cast<T*>(p.context);
    if (from_tile >= to_tile) {
        if (tiles == 0 && number == 0) {  // a row that sees nothing
            for (int i = threadIdx.x; i < rows * head_dim; i += kThreads) context[element_of(i / head_dim) + i % head_dim] = from_float<T>(0.0f);
        }
        return;
    }
    const int32_t* pages = t.pages + (int64_t)row * t.max_pages;
    const int64_t row_bytes = (int64_t)head_dim * sizeof(T), head_bytes = row_bytes * t.page_size, page_bytes = head_bytes * kv_heads;
    const char* keys = p.cache.keys + head * head_bytes;
    const int64_t apart = p.cache.values - p.cache.keys;
    const auto page_of = [&](int tile) { return tile < to_tile ? pages[(tile0 + tile) * kTile >> t.shift] : -1; };
    int page = page_of(from_tile + warp), next_page = page_of(from_tile + warp + kWarps);

    // The query rows as the right-hand operand, in shared memory: for each step of two products, by (tile of rows, step, product, lane), the words
    // of row gid that lane (gid, tig) wants; fp32's in two parts.  The warps share the work.
    using Words = typename std::conditional<precise, uint4, uint2>::type;
    Words* parts = reinterpret_cast<Words*>(shared);
    for (int i = warp; i < tiles_of_rows * kSteps; i += kWarps) {
        const int r = i / kSteps * 8 + gid, d = i % kSteps * 4 * E + tig * E;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && d < head_dim) x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + element_of(r) + d);
        if constexpr (precise) {
            const uint32_t h[4] = {eleven_bits(x.x), eleven_bits(x.y), eleven_bits(x.z), eleven_bits(x.w)};
            parts[2 * i * 32 + lane] = make_uint4(h[0], h[1], left_of(x.x, h[0]), left_of(x.y, h[1]));
            parts[(2 * i + 1) * 32 + lane] = make_uint4(h[2], h[3], left_of(x.z, h[2]), left_of(x.w, h[3]));
        } else {
            parts[2 * i * 32 + lane] = make_uint2(x.x, x.y);
            parts[(2 * i + 1) * 32 + lane] = make_uint2(x.z, x.w);
        }
    }
    __syncthreads();

    float out[tiles_of_rows][kBlocks][4], top[tiles_of_rows][2], total[tiles_of_rows][2];
    int first[tiles_of_rows][2], last[tiles_of_rows][2];
#pragma unroll
    for (int n = 0; n < tiles_of_rows; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[n][i] = kNone, total[n][i] = 0.0f;
            const int own = min((first_row + n * 8 + 2 * tig + i) / p.group, p.q_len - 1);
            first[n][i] = sight.first(own), last[n][i] = sight.last(own, p.causal != 0);
        }
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) out[n][m][0] = out[n][m][1] = out[n][m][2] = out[n][m][3] = 0.0f;
    }
    const int seen = max(sight.first(0), 0);                                               // no row sees a position before this one
    const int all_from = sight.first(p.q_len - 1), all_to = sight.last(0, p.causal != 0);  // every row sees those between
    const float factor = p.scale * kLog2e;

    // A tile, and where its positions lie.  What no row sees, and pages that are none, arrive as zeros, whatever lies there.
    struct Place {
        int position;
        bool real, whole, plain;  // its page is one of the pool; all of its positions are seen by some row; and its rows are as long as the kernel's
        const char* keys;
    };
    const auto place_of = [&](int tile, int page) {
        Place at;
        at.position = (tile0 + tile) * kTile;
        at.real = t.real(page);  // (a tile that is not there has the page -1)
        at.whole = at.real && at.position >= seen && at.position + kTile <= length;
        at.plain = at.whole && head_dim == dims;
        at.keys = keys + (at.real ? page : 0) * page_bytes + (at.position & (t.page_size - 1)) * row_bytes;
        return at;
    };
    const auto there = [&](const Place& at, int r) { return at.whole || (at.real && at.position + r >= seen && at.position + r < length); };
    uint4 k[kSegment][2], v[kBlocks / K::tiles][4];
    const auto load_keys = [&](const Place& place, int s0) {
        if (place.plain) {  // (one address, and distances that are known)
            const char* at = place.keys + (gid * dims + tig * E) * (int)sizeof(T);
#pragma unroll
            for (int s = 0; s < kSegment; ++s) {
                k[s][0] = load_once(at + (s0 + s) * 4 * E * (int)sizeof(T));
                k[s][1] = load_once(at + (8 * dims + (s0 + s) * 4 * E) * (int)sizeof(T));
            }
        } else {
            const bool low_there = there(place, gid), high_there = there(place, gid + 8);
#pragma unroll
            for (int s = 0; s < kSegment; ++s) {
                const int d = (s0 + s) * 4 * E + tig * E;
                k[s][0] = k[s][1] = make_uint4(0, 0, 0, 0);
                if (low_there && d < head_dim) k[s][0] = load_once(place.keys + gid * row_bytes + d * (int)sizeof(T));
                if (high_there && d < head_dim) k[s][1] = load_once(place.keys + (gid + 8) * row_bytes + d * (int)sizeof(T));
            }
        }
    };
    const auto load_values = [&](const Place& place) {
        if (place.plain) {
            const char* at = place.keys + apart + ((precise ? tig : 2 * tig) * dims + gid * E) * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int m = 0; m < kBlocks / K::tiles; ++m) {
                    v[m][i] = load_once(at + ((precise ? 4 * i : (i & 1) + (i >> 1) * 8) * dims + m * 8 * E) * (int)sizeof(T));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = precise ? tig + 4 * i : 2 * tig + (i & 1) + (i >> 1) * 8;
                const bool real_row = there(place, r);
#pragma unroll
                for (int m = 0; m < kBlocks / K::tiles; ++m) {
                    const int d = m * 8 * E + gid * E;
                    v[m][i] = make_uint4(0, 0, 0, 0);
                    if (real_row && d < head_dim) v[m][i] = load_once(place.keys + apart + r * row_bytes + d * (int)sizeof(T));
                }
            }
        }
    };
    Place now = place_of(from_tile + warp, page);
    if (keys_ahead) load_keys(now, 0);
    for (int tile = from_tile + warp; tile < to_tile; tile += kWarps) {
        const Place next = place_of(tile + kWarps, next_page);
        next_page = page_of(tile + 2 * kWarps);
        const int position = now.position;
        const bool real = now.real;
        if (keys_ahead) load_values(now);
        float score[tiles_of_rows][4];
#pragma unroll
        for (int n = 0; n < tiles_of_rows; ++n) score[n][0] = score[n][1] = score[n][2] = score[n][3] = 0.0f;
#pragma unroll
        for (int s0 = 0; s0 < kSteps; s0 += kSegment) {
            if (!keys_ahead) load_keys(now, s0);
#pragma unroll
            for (int s = 0; s < kSegment; ++s) {
                const uint32_t a[2][4] = {{k[s][0].x, k[s][1].x, k[s][0].y, k[s][1].y}, {k[s][0].z, k[s][1].z, k[s][0].w, k[s][1].w}};
#pragma unroll
                for (int n = 0; n < tiles_of_rows; ++n) {
                    if constexpr (precise) {
                        float some[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int j = 0; j < 2; ++j) multiply_parts(some, a[j], parts[((n * kSteps + s0 + s) * 2 + j) * 32 + lane]);
                        add_to(score[n], some);
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const Words q = parts[((n * kSteps + s0 + s) * 2 + j) * 32 + lane];
                            multiply(score[n], a[j], q.x, q.y, T{});
                        }
                    }
                }
            }
        }
        if (keys_ahead) load_keys(next, 0);
        else load_values(now);
        now = next;
        // score[n][2 o + i]: position 8 o + gid, query row 8 n + 2 tig + i
        const bool masked = !real || position < all_from || position + kTile - 1 > all_to;
#pragma unroll
        for (int n = 0; n < tiles_of_rows; ++n) {
            float high[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const int j = position + 8 * o + gid;
                    score[n][2 * o + i] *= factor;
                    if (masked && (!real || j < first[n][i] || j > last[n][i])) score[n][2 * o + i] = kNone;
                }
                high[i] = fmaxf(score[n][i], score[n][2 + i]) - K::lift;
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
        // Weights, turned round: lane (gid, tig) then holds query row gid's weights of the positions whose values it has.
        uint32_t wh[tiles_of_rows][2][2], wl[tiles_of_rows][2][2];
#pragma unroll
        for (int n = 0; n < tiles_of_rows; ++n) {
            const float t0 = top[n][0] > kNone ? top[n][0] : 0.0f, t1 = top[n][1] > kNone ? top[n][1] : 0.0f;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const float w0 = exp2_approx(score[n][2 * o] - t0), w1 = exp2_approx(score[n][2 * o + 1] - t1);
                total[n][0] += w0;
                total[n][1] += w1;
                if constexpr (precise) {
                    // lane (gid, tig) wants row gid's weights of positions 8 o + tig and 8 o + tig + 4: they are in lanes (tig, gid / 2) and
                    // (tig + 4, gid / 2), in the first place for even rows, in the second for odd ones
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int from = (tig + 4 * i) * 4 + gid / 2;
                        const float even = __shfl_sync(0xffffffffu, w0, from), odd = __shfl_sync(0xffffffffu, w1, from);
                        const uint32_t w = __float_as_uint(gid & 1 ? odd : even);
                        wh[n][o][i] = eleven_bits(w);
                        wl[n][o][i] = left_of(w, wh[n][o][i]);
                    }
                } else {
                    const uint32_t taken = pair_of<T>(w0, w1);
                    wh[n][0][o] = transposed(taken);
                    wl[n][0][o] = transposed(pair_left<T>(w0, w1, taken));
                }
            }
        }
#pragma unroll
        for (int m = 0; m < kBlocks / K::tiles; ++m) {
            const uint32_t x[4][4] = {{v[m][0].x, v[m][0].y, v[m][0].z, v[m][0].w}, {v[m][1].x, v[m][1].y, v[m][1].z, v[m][1].w},
                                      {v[m][2].x, v[m][2].y, v[m][2].z, v[m][2].w}, {v[m][3].x, v[m][3].y, v[m][3].z, v[m][3].w}};
#pragma unroll
            for (int i = 0; i < K::tiles; ++i) {
                if constexpr (precise) {
                    float some[tiles_of_rows][4] = {};
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        const uint32_t a[4] = {x[2 * o][2 * i], x[2 * o][2 * i + 1], x[2 * o + 1][2 * i], x[2 * o + 1][2 * i + 1]};
#pragma unroll
                        for (int n = 0; n < tiles_of_rows; ++n) {
                            multiply_parts(some[n], a, make_uint4(wh[n][o][0], wh[n][o][1], wl[n][o][0], wl[n][o][1]));
                        }
                    }
#pragma unroll
                    for (int n = 0; n < tiles_of_rows; ++n) add_to(out[n][m * K::tiles + i], some[n]);
                } else {
                    const uint32_t a[4] = {__byte_perm(x[0][i], x[1][i], 0x5410), __byte_perm(x[0][i], x[1][i], 0x7632),
                                           __byte_perm(x[2][i], x[3][i], 0x5410), __byte_perm(x[2][i], x[3][i], 0x7632)};
#pragma unroll
                    for (int n = 0; n < tiles_of_rows; ++n) {
                        multiply(out[n][m * K::tiles + i], a, wl[n][0][0], wl[n][0][1], T{});
                        multiply(out[n][m * K::tiles + i], a, wh[n][0][0], wh[n][0][1], T{});
                    }
                }
            }
        }
    }

    // The four warps' results meet in shared memory.
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
            const int d = m / K::tiles * 8 * E + gid * E + m % K::tiles * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *reinterpret_cast<float2*>(meet + (warp * kRows + n * 8 + 2 * tig + i) * dims + d) = make_float2(out[n][m][i], out[n][m][2 + i]);
            }
        }
    }
    __syncthreads();
    // What makes a row's weights add up to one.  A sum of 0: the row sees nothing, or (as in any softmax, NaN) scores of -inf alone.
    const auto inverse_of = [&](int r, float sum) {
        if (sum != 0.0f) return 1.0f / sum;
        const int own = (first_row + r) / p.group;
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
            store_four(context + element_of(r) + d, value, inverse_of(r, sum));
        } else {
            __stcg(reinterpret_cast<float4*>(piece + r * (dims + 4) + d), value);
            if (d == 0) __stcg(reinterpret_cast<float2*>(piece + r * (dims + 4) + dims), make_float2(high, sum));
        }
    }
    if (whole) return;
    const int pieces = (tiles + share - 1) / share;
    __syncthreads();
    if (threadIdx.x == 0) {  // (release: the block's pieces, ordered before by the barrier; acquire: the other blocks')
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + unit) : "memory");
        is_last = before == pieces - 1;
        if (is_last) p.arrived[unit] = 0;
    }
    __syncthreads();
    if (!is_last) return;
    const auto piece_of = [&](int b) { return p.partial + ((int64_t)unit * p.pieces + b) * piece_floats; };
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
            const float weight = mine.x > kNone ? exp2_approx(mine.x - high) : 0.0f;
            less[b * rows + r].x = weight;
            sum += weight * mine.y;
        }
#pragma unroll
        for (int step = 16; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
        if (lane == 0) totals[0][r] = sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * fours; i += kThreads) {
        const int r = i / fours, d = i % fours * 4;
        float4 value = make_float4(0, 0, 0, 0);
        const auto add = [&](const float4& part, float weight) {
            value.x += part.x * weight, value.y += part.y * weight, value.z += part.z * weight, value.w += part.w * weight;
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
        store_four(context + element_of(r) + d, value, inverse_of(r, totals[0][r]));
    }
}

int padded_dims(const PagedAttentionParams& p) { return p.cache.head_dim > 128 ? 256 : p.cache.head_dim > 64 ? 128 : 64; }
int tiles_of_rows(const PagedAttentionParams& p) { return p.rows <= 8 || padded_dims(p) == 256 ? 1 : 2; }  // (of a block's kernel)

template <class T, int dims, int tiles_of_rows>
cudaError_t launch(const PagedAttentionParams& p, cudaStream_t stream) {
    constexpr size_t shared = shared_of(dims, tiles_of_rows, sizeof(T) == 4);
    void (*const kernel)(const PagedAttentionParams) = decode_attention_pages_kernel<T, dims, tiles_of_rows>;
    static_assert(shared <= 40 << 10, "more than a kernel gets unasked");
    return launch_overlapping(kernel, dim3((unsigned)(paged_attention_counters(p) * p.pieces)), dim3(kThreads), shared, stream, p);
}

template <class T>
cudaError_t launch_type(const PagedAttentionParams& p, cudaStream_t stream) {
    const int dims = padded_dims(p);
    if (dims == 256) return launch<T, 256, 1>(p, stream);
    if (tiles_of_rows(p) == 1) return dims == 128 ? launch<T, 128, 1>(p, stream) : launch<T, 64, 1>(p, stream);
    return dims == 128 ? launch<T, 128, 2>(p, stream) : launch<T, 64, 2>(p, stream);
}

}  // namespace

void plan_paged_attention(PagedAttentionParams& p, int sm_count) {
    const int dims = padded_dims(p), width = element_bytes(p.type);
    p.row_groups = dims == 256 ? (p.rows + 7) / 8 : 1;  // (more rows' contexts do not fit the registers; the cache comes out of L2 the second time)
    const int64_t tiles = (p.cache.table.capacity() + kTile - 1) / kTile, units = paged_attention_counters(p);
    // Blocks that the GPU holds at once.
    const int64_t blocks = (int64_t)sm_count * blocks_of(dims, width, tiles_of_rows(p));
    // The pieces of a pair have their maxima and sums in shared memory when they are joined.
    const int64_t most = std::min<int64_t>((tiles + kWarps - 1) / kWarps, shared_of(dims, tiles_of_rows(p), width == 4) / (8 * tiles_of_rows(p) * sizeof(float2)));
    const int64_t spread = std::max<int64_t>(1, std::min(blocks / units, (int64_t)std::sqrt(kSplitRate * tiles)));
    const int64_t balanced = std::min((tiles + most_share(dims) - 1) / most_share(dims), 16 * blocks / units);  // (blocks that find nothing to do cost time too)
    p.spread = (int)std::min(spread, most);
    p.pieces = (int)std::min(std::max(spread, balanced), most);
}

int64_t paged_attention_counters(const PagedAttentionParams& p) { return (int64_t)p.cache.table.rows * p.cache.kv_heads * p.row_groups; }

size_t paged_attention_partial_bytes(const PagedAttentionParams& p) {
    return (size_t)(paged_attention_counters(p) * p.pieces) * 8 * tiles_of_rows(p) * (padded_dims(p) + 4) * sizeof(float);
}

cudaError_t launch_paged_attention(const PagedAttentionParams& p, cudaStream_t stream) {
    if (p.rows > 16 || p.cache.head_dim > 256) return cudaErrorInvalidValue;
    if (p.type == kFloat32) return launch_type<float>(p, stream);
    if (p.type == kBfloat16) return launch_type<__nv_bfloat16>(p, stream);
    return launch_type<__half>(p, stream);
}

}  // namespace psx
