// Log-probabilities of given tokens, with the entropy of the row and its largest alternatives, in one pass over the logits.
//
// With m the row's largest logit and sums over all logits but one that is m,
//     r = sum exp(x - m),   log p(t) = (x_t - m) - log(1 + r),   H = log(1 + r) + sum (m - x) exp(x - m) / (1 + r).
// The largest itself stays out of the sums, so that a row whose token is nearly certain has the digits of r = 1e-9 and not those of 1 + r: a
// thread keeps the largest of its logits aside, and whatever is not larger than it (or the one that it replaces) joins the sums, relative to
// the thread's largest so far.  16-bit logits are compared in pairs as they come.
//
// A block takes a part of a row, in chunks of up to 16 vectors of 16 bytes per thread, the next one on its way; the part leaves m, its two sums
// and its `top` best logits in order.  They are found as beam_select.cu finds them: a bound that at least `top` logits reach from the
// threads' largest, a second look, out of L2, at the few chunks that reach it, and an entry's place is the number of keys above its own.  The block
// of a row that ends last goes on with the row.  Rows need not be aligned: vectors are those of memory, and where one is cut by an end of the row its
// elements are read one by one.  Bound by HBM: the logits, once.
#include "token_log_probs.cuh"

#include <algorithm>
#include <type_traits>

#include "row_selection.cuh"

namespace psx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostChunks = 8;  // of a part
constexpr int kLongVectors = 4;
constexpr int kPartList = 1024, kRowList = 1024;
constexpr int kHeldEntries = 8;  // per thread, of the parts' lists
constexpr float kLeast = -200.0f;  // 2^-200 is 0 as a float; the logarithm of a weight is never less (0 times -inf would be NaN)
constexpr int kRowOk = 0, kRowNonFinite = 4, kRowAllRemoved = 5, kRowBadToken = 66;  // (psx_row_status)

// NaN where one of the two is.
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float smaller(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// (In the order of integers, ordered() and from_ordered(), a warp's maximum passed over a NaN although its integer is the largest: 31 of a NaN and 1 to 31.)
__device__ __forceinline__ float warp_largest(float x) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

// A word of a vector: one float or two 16-bit numbers.
template <class T>
struct Word {
    static constexpr int elements = 4 / sizeof(T);
    uint32_t bits;

    __device__ __forceinline__ static Word none() {
        if constexpr (sizeof(T) == 4) return {0xff800000u};
        else return {std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u};
    }
    __device__ __forceinline__ float2 floats() const {
        if constexpr (sizeof(T) == 4) {
            return make_float2(__uint_as_float(bits), kNone);
        } else if constexpr (std::is_same<T, __half>::value) {
            __half2 h;
            __builtin_memcpy(&h, &bits, 4);
            return __half22float2(h);
        } else {
            return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
        }
    }
    __device__ __forceinline__ Word max_with(Word o) const {
        Word r;
        if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        else if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        return r;
    }
    __device__ __forceinline__ Word min_with(Word o) const {
        Word r;
        if constexpr (sizeof(T) == 4) asm("min.NaN.f32 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        else if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r.bits) : "r"(bits), "r"(o.bits));
        return r;
    }
};

struct PartShared {
    uint64_t list[kPartList], best_of[kWarps];
    uint32_t bounds[kWarps];
    float tops[kWarps], sums[kWarps], weighted[kWarps];
    int listed;
};

// Of several holders of (m, sums), all lanes of a warp taking part: the sums relative to `high`, the largest m, of which `first` is one holder.
__device__ __forceinline__ void relative_to(float high, bool first, float m, float& sum, float& weighted) {
    if (first) return;
    const float y = fmaxf((m - high) * kLog2e, kLeast), f = m > kNone ? exp2_approx(y) : 0.0f;
    weighted = (weighted + y * (1.0f + sum)) * f;
    sum = (1.0f + sum) * f;
}

template <class T, int vectors, bool picks>
__device__ __forceinline__ void part_of_row(const TokenLogProbsParams& p, PartShared& s) {
    constexpr int E = 16 / sizeof(T), kChunk = kThreads * vectors * E, kWords = vectors * 4;
    using W = Word<T>;
    const int64_t part_row = blockIdx.x;
    const int64_t row = part_row / p.parts;
    const int part = (int)(part_row % p.parts), warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) s.listed = 0;
    // Elements are counted from the 16-byte boundary that is not behind the row's first one.
    const T* from = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int shift = (int)(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
    from -= shift;
    const int64_t all = (int64_t)shift + p.vocab;
    const int64_t begin = (int64_t)part * p.chunks * kChunk, end = min(begin + (int64_t)p.chunks * kChunk, all);
    const auto column = [&](int chunk, int v) { return begin + (int64_t)chunk * kChunk + (v * kThreads + (int)threadIdx.x) * E; };
    const auto load = [&](int chunk, W (&w)[kWords], bool again) {
#pragma unroll
        for (int v = 0; v < vectors; ++v) {
            const int64_t at = column(chunk, v);
            uint4 x = make_uint4(W::none().bits, W::none().bits, W::none().bits, W::none().bits);
            if (at >= shift && at + E <= end) {
                x = again ? __ldcg(reinterpret_cast<const uint4*>(from + at)) : __ldcs(reinterpret_cast<const uint4*>(from + at));
            } else if (at < end && at + E > shift) {  // (an end of the row)
                T e[E];
                __builtin_memcpy(e, &x, 16);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (at + i >= shift && at + i < end) e[i] = from[at + i];
                }
                __builtin_memcpy(&x, e, 16);
            }
            w[4 * v].bits = x.x, w[4 * v + 1].bits = x.y, w[4 * v + 2].bits = x.z, w[4 * v + 3].bits = x.w;
        }
    };

    W w[2][kWords], best = W::none();  // (best: the largest so far, of even and of odd places for 16-bit logits)
    float chunk_top[picks ? kMostChunks : 1], level = kNone;
    float2 sum = {0.0f, 0.0f}, weighted = {0.0f, 0.0f};
    load(0, w[0], false);
#pragma unroll
    for (int c = 0; c < kMostChunks; ++c) {
        if constexpr (picks) chunk_top[c] = kNone;
        if (c < p.chunks) {
            if (c + 1 < kMostChunks && c + 1 < p.chunks) load(c + 1, w[(c + 1) % 2], false);
            W(&x)[kWords] = w[c % 2];
            if constexpr (picks) {
                W high[2] = {x[0], x[1]};
#pragma unroll
                for (int i = 2; i < kWords; ++i) high[i % 2] = high[i % 2].max_with(x[i]);
                const float2 two = high[0].max_with(high[1]).floats();
                chunk_top[c] = larger(two.x, two.y);
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {  // the larger one is kept aside
                const W lower = best.min_with(x[i]);
                best = best.max_with(x[i]);
                x[i] = lower;
            }
            const float2 two = best.floats();
            const float next = fmaxf(two.x, two.y), base = next > kNone ? next : 0.0f;
            const float less = fmaxf((level - base) * kLog2e, kLeast), factor = exp2_approx(less);
            weighted = mul_pair(fma_pair(make_float2(less, less), sum, weighted), make_float2(factor, factor));
            sum = mul_pair(sum, make_float2(factor, factor));
            level = base;
            const float2 minus = make_float2(-base, -base), log2e = make_float2(kLog2e, kLog2e);
#pragma unroll
            for (int i = 0; i < kWords; i += W::elements == 1 ? 2 : 1) {
                float2 y = x[i].floats();
                if constexpr (W::elements == 1) y.y = x[i + 1].floats().x;
                y = mul_pair(add_pair(y, minus), log2e);
                y = make_float2(fmaxf(y.x, kLeast), fmaxf(y.y, kLeast));
                const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                sum = add_pair(sum, e);
                weighted = fma_pair(y, e, weighted);
            }
        }
    }
    // The thread's own: the smaller of the two that are aside joins the sums.
    const float2 aside = best.floats();
    const float top = larger(aside.x, aside.y);
    float own = sum.x + sum.y, own_weighted = weighted.x + weighted.y;
    if constexpr (W::elements == 2) {
        const float y = fmaxf((smaller(aside.x, aside.y) - level) * kLog2e, kLeast), e = exp2_approx(y);
        own += e;
        own_weighted += y * e;
    }
    const float warp_top = warp_largest(top);
    const unsigned holders = __ballot_sync(0xffffffffu, top == warp_top);
    relative_to(warp_top, lane == __ffs(holders) - 1, top, own, own_weighted);
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
        own += __shfl_xor_sync(0xffffffffu, own, step);
        own_weighted += __shfl_xor_sync(0xffffffffu, own_weighted, step);
    }
    uint32_t mine = 0;
    if constexpr (picks) mine = warp_bound<kWarps>(top, p.top, nullptr);
    if (lane == 0) s.bounds[warp] = mine, s.tops[warp] = warp_top, s.sums[warp] = own, s.weighted[warp] = own_weighted;
    __syncthreads();
    if (warp == kWarps - 1) {  // the part's record
        const float m = lane < kWarps ? s.tops[lane] : kNone;
        const float high = warp_largest(m);
        float part_sum = lane < kWarps ? s.sums[lane] : 0.0f, part_weighted = lane < kWarps ? s.weighted[lane] : 0.0f;
        const unsigned holds = __ballot_sync(0xffffffffu, lane < kWarps && m == high);
        relative_to(high, lane == __ffs(holds) - 1, m, part_sum, part_weighted);
#pragma unroll
        for (int step = 4; step > 0; step /= 2) {
            part_sum += __shfl_xor_sync(0xffffffffu, part_sum, step);
            part_weighted += __shfl_xor_sync(0xffffffffu, part_weighted, step);
        }
        if (lane == 0) __stcg(reinterpret_cast<float4*>(p.stats + part_row), make_float4(high, part_sum, part_weighted, 0.0f));
    }
    if constexpr (picks) {
        const int keep = p.top;
        LogProbEntry* entries = p.entries + part_row * keep;
        const auto put = [&](int place, uint64_t key) {
            __stcg(reinterpret_cast<float2*>(entries + place), make_float2(from_ordered((uint32_t)(key >> 32)), __int_as_float((int)~(uint32_t)key)));
        };
        uint32_t bound_key = s.bounds[0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) bound_key = min(bound_key, s.bounds[i]);
        const float bound = bound_key == 0 ? kNone : from_ordered(bound_key);
        uint32_t hits = 0;  // the chunks that reach the bound; they are read again, out of L2
#pragma unroll
        for (int c = 0; c < kMostChunks; ++c) hits |= (chunk_top[c] >= bound && chunk_top[c] > kNone) ? 1u << c : 0u;
        // every logit of those chunks that reaches the bound, with its token
        const auto look = [&](auto take) {
            for (uint32_t rest = hits; rest != 0; rest &= rest - 1) {
                const int c = __ffs(rest) - 1;
                load(c, w[0], true);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const float2 x = w[0][i].floats();
                    const int token = (int)(column(c, i / 4) - shift) + i % 4 * W::elements;
                    if (x.x >= bound && x.x > kNone) take(x.x, token);
                    if constexpr (W::elements == 2) {
                        if (x.y >= bound && x.y > kNone) take(x.y, token + 1);
                    }
                }
            }
        };
        look([&](float x, int token) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < kPartList) s.list[at] = entry_key(x, token);
        });
        __syncthreads();
        const int count = s.listed;
        int placed = min(count, keep);
        if (count <= kPartList) {
            for (int e = threadIdx.x; e < count; e += kThreads) {
                const uint64_t key = s.list[e];
                int place = 0;
#pragma unroll 4
                for (int k = 0; k < count; ++k) place += s.list[k] > key;
                if (place < keep) put(place, key);
            }
        } else {  // (thousands that tie at the bound)
            uint64_t last = ~0ull;
            for (placed = 0; placed < keep; ++placed) {
                uint64_t next = 0;
                look([&](float x, int token) {
                    const uint64_t key = entry_key(x, token);
                    if (key < last) next = max(next, key);
                });
                next = block_max<kWarps>(next, s.best_of);
                if (next == 0) break;
                if (threadIdx.x == 0) put(placed, next);
                last = next;
            }
        }
        for (int i = placed + threadIdx.x; i < keep; i += kThreads) __stcg(reinterpret_cast<float2*>(entries + i), make_float2(kNone, __int_as_float(-1)));
    }
}

struct RowShared {
    uint64_t list[kRowList], best_of[kWarps];
    uint32_t bounds[kWarps];
    double top, lse;  // the row's largest logit and log(1 + r)
    int listed, status;
};

// What the parts' blocks have written: out of L2.
__device__ __forceinline__ uint64_t key_of(const LogProbEntry* at) {
    const float2 two = __ldcg(reinterpret_cast<const float2*>(at));
    return two.x > kNone ? entry_key(two.x, __float_as_int(two.y)) : 0;
}

template <class T, bool picks>
__device__ __forceinline__ void whole_row(const TokenLogProbsParams& p, RowShared& s, int64_t row) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, parts = p.parts, keep = p.top;
    const LogProbEntry* entries = p.entries + row * parts * keep;
    // The lists' first entries, then the second ones and so on, are asked for ahead of the sums and kept; neighbours go to different warps.
    uint64_t held[kHeldEntries];
    constexpr int kHeld = kHeldEntries * kThreads;
    if constexpr (picks) {
        if (threadIdx.x == 0) s.listed = 0;
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) {
            const int x = i * kThreads + lane * kWarps + warp;
            held[i] = x < parts * keep ? key_of(entries + (int64_t)(x % parts) * keep + x / parts) : 0;
        }
    }
    if (warp == 0) {
        const float4* stats = reinterpret_cast<const float4*>(p.stats + row * parts);
        const int64_t token = p.tokens ? p.tokens[row] : 0;
        const bool real = token >= 0 && token < p.vocab;
        float logit = 0.0f;
        if (p.tokens && real && lane == 0) logit = to_float(static_cast<const T*>(p.logits)[row * p.row_stride + token]);
        float high = kNone;
        for (int i = lane; i < parts; i += 32) high = larger(high, __ldcg(stats + i).x);
        high = warp_largest(high);
        const bool wrong = !(high < -kNone), none = high == kNone;
        double r = 0.0, weighted = 0.0;
        bool found = false;  // the part that holds the row's largest, the first of them
        for (int first = 0; first < parts; first += 32) {
            const int i = first + lane;
            const float4 x = i < parts ? __ldcg(stats + i) : make_float4(kNone, 0.0f, 0.0f, 0.0f);
            const unsigned holders = __ballot_sync(0xffffffffu, x.x == high);
            float sum = x.y, w = x.z;
            relative_to(high, !found && lane == __ffs(holders) - 1, x.x, sum, w);
            found |= holders != 0;
            r += sum;
            weighted += w;
        }
#pragma unroll
        for (int step = 16; step > 0; step /= 2) {
            r += __shfl_xor_sync(0xffffffffu, r, step);
            weighted += __shfl_xor_sync(0xffffffffu, weighted, step);
        }
        if (lane == 0) {
            const double lse = log_of_one_and(r);
            const float nan = __int_as_float(0x7fffffff);
            s.top = high;
            s.lse = lse;
            s.status = wrong ? kRowNonFinite : none ? kRowAllRemoved : p.tokens && !real ? kRowBadToken : kRowOk;
            if (p.tokens) p.log_probs[row] = wrong || none || !real ? nan : (float)(((double)logit - (double)high) - lse);
            if (p.entropy) p.entropy[row] = wrong || none ? nan : (float)(lse - weighted * 0.69314718055994530942 / (1.0 + r));
            if (p.row_status) p.row_status[row] = s.status;
        }
    }
    if constexpr (picks) {
        uint64_t largest = 0;
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) largest = max(largest, held[i]);
        const uint32_t mine = warp_bound<kWarps>(largest ? from_ordered((uint32_t)(largest >> 32)) : kNone, keep, nullptr);
        if (lane == 0) s.bounds[warp] = mine;
        __syncthreads();
        uint32_t bound = s.bounds[0];
        for (int w = 1; w < kWarps; ++w) bound = min(bound, s.bounds[w]);
        const auto offer = [&](uint64_t key) {
            if (key == 0 || (uint32_t)(key >> 32) < bound) return false;
            const int at = atomicAdd(&s.listed, 1);
            if (at < kRowList) s.list[at] = key;
            return true;
        };
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) offer(held[i]);
        if (kHeld < parts * keep) {  // lists are in order: each from where it is not held on, as far as it reaches the bound
            for (int q = threadIdx.x; q < parts; q += kThreads) {
                for (int slot = max(kHeld - q + parts - 1, 0) / parts; slot < keep && offer(key_of(entries + (int64_t)q * keep + slot)); ++slot) {
                }
            }
        }
        __syncthreads();
        const int count = s.listed;
        const bool wrong = s.status == kRowNonFinite;
        int placed = wrong ? 0 : min(count, keep);
        const auto put = [&](int place, uint64_t key) {
            p.top_log_probs[row * keep + place] = (float)(((double)from_ordered((uint32_t)(key >> 32)) - s.top) - s.lse);
            p.top_tokens[row * keep + place] = (int64_t)~(uint32_t)key;
        };
        if (wrong) {
        } else if (count <= kRowList) {
            for (int e = threadIdx.x; e < count; e += kThreads) {
                const uint64_t key = s.list[e];
                int place = 0;
#pragma unroll 4
                for (int k = 0; k < count; ++k) place += s.list[k] > key;
                if (place < keep) put(place, key);
            }
        } else {  // more that tie at the bound than the list holds: sweep after sweep, the best that is behind the last one
            uint64_t last = ~0ull;
            for (placed = 0; placed < keep; ++placed) {
                uint64_t next = 0;
                for (int64_t e = threadIdx.x; e < (int64_t)parts * keep; e += kThreads) {
                    const uint64_t key = key_of(entries + e);
                    if (key < last) next = max(next, key);
                }
                next = block_max<kWarps>(next, s.best_of);
                if (next == 0) break;
                if (threadIdx.x == 0) put(placed, next);
                last = next;
            }
        }
        for (int i = placed + threadIdx.x; i < keep; i += kThreads) {
            p.top_log_probs[row * keep + i] = wrong ? __int_as_float(0x7fffffff) : kNone;
            p.top_tokens[row * keep + i] = -1;
        }
    }
}

template <class T, int vectors, bool picks>
__global__ void __launch_bounds__(kThreads, vectors == 1 ? 2 : 4) token_log_probs_kernel(const __grid_constant__ TokenLogProbsParams p) {
    __shared__ union Shared {
        PartShared part;
        RowShared row;
        __device__ Shared() {}
    } shared;
    __shared__ int is_last;
    part_of_row<T, vectors, picks>(p, shared.part);
    const int64_t row = blockIdx.x / (unsigned)p.parts;
    __syncthreads();
    if (p.parts > 1) {
        if (threadIdx.x == 0) {  // (release: the block's part, ordered before by the barrier; acquire: the others')
            int before;
            asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + row) : "memory");
            is_last = before == p.parts - 1;
            if (is_last) p.arrived[row] = 0;
        }
        __syncthreads();
        if (!is_last) return;
    }
    whole_row<T, picks>(p, shared.row, row);
}

template <class T>
cudaError_t launch_type(const TokenLogProbsParams& p, cudaStream_t stream) {
    const unsigned blocks = (unsigned)(p.rows * p.parts);
    if (p.vectors == 1) {
        if (p.top > 0) token_log_probs_kernel<T, 1, true><<<blocks, kThreads, 0, stream>>>(p);
        else token_log_probs_kernel<T, 1, false><<<blocks, kThreads, 0, stream>>>(p);
    } else {
        if (p.top > 0) token_log_probs_kernel<T, kLongVectors, true><<<blocks, kThreads, 0, stream>>>(p);
        else token_log_probs_kernel<T, kLongVectors, false><<<blocks, kThreads, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace

void plan_token_log_probs(TokenLogProbsParams& p, int sm_count) {
    const int E = 16 / element_bytes(p.type);
    // Long parts cost least per logit (what a part costs besides is shared by up to eight chunks); where they would be fewer than the
    // GPU holds at once, shorter ones spread the rows further.
    const auto chunks = [&](int vectors) { return ((int64_t)p.vocab + E - 1 + kThreads * vectors * E - 1) / (kThreads * vectors * E); };
    p.vectors = p.rows * chunks(kLongVectors) < sm_count ? 1 : kLongVectors;
    const int64_t all = chunks(p.vectors);
    p.chunks = kMostChunks;
    while (p.chunks > 1 && p.rows * ((all + p.chunks - 1) / p.chunks) < 2 * sm_count) --p.chunks;
    p.parts = (int)((all + p.chunks - 1) / p.chunks);
    p.chunks = (int)((all + p.parts - 1) / p.parts);  // (no part much shorter than the others)
}

cudaError_t launch_token_log_probs(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.type == kFloat32) return launch_type<float>(p, stream);
    if (p.type == kBfloat16) return launch_type<__nv_bfloat16>(p, stream);
    return launch_type<__half>(p, stream);
}

}  // namespace psx
