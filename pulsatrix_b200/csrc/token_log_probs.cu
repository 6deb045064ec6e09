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
constexpr int kMostChunks = 32;  // of a part
constexpr int kLongVectors = 4;
constexpr int kBlocks = 4;  // that an SM holds
constexpr int kMostMaxima = (kMostTop + kWarps - 1) / kWarps + 2;  // of a warp
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
    static constexpr float lowest = std::is_same<T, __half>::value ? -65504.0f : -0x1.fep127f;
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
    // Both numbers and `minus`, as floats.
    __device__ __forceinline__ float2 plus(float minus) const {
        float2 r;
        if constexpr (sizeof(T) == 4) r = make_float2(__uint_as_float(bits) + minus, kNone);
        else if constexpr (std::is_same<T, __half>::value)
            asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %3;\n\tadd.rn.f32.f16 %1, h, %3;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(bits), "f"(minus));
        else
            asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.bf16 %0, l, %3;\n\tadd.rn.f32.bf16 %1, h, %3;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(bits), "f"(minus));
        return r;
    }
    __device__ __forceinline__ static Word both(float x) {  // rounded
        if constexpr (sizeof(T) == 4) return {__float_as_uint(x)};
        const T two[2] = {from_float<T>(x), from_float<T>(x)};
        Word r;
        __builtin_memcpy(&r.bits, two, 4);
        return r;
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

// A bound that at least `keep` of the block's numbers reach, each thread giving its largest: the `keep`-th largest of what the warps' largest few make
// (two more than an equal share; where one warp has more of the largest than that the bound is lower than it could be), 0 where there are not so many.
__device__ __forceinline__ int maxima_of(int keep) { return (keep + kWarps - 1) / kWarps + (keep > 1 ? 2 : 0); }
__device__ __forceinline__ void warp_maxima(float largest, int keep, uint32_t* maxima) {
    const int each = maxima_of(keep), lane = threadIdx.x % 32;
    uint32_t key = largest > kNone ? ordered(largest) : 0;
    for (int i = 0; i < each;) {
        const uint32_t next = __reduce_max_sync(0xffffffffu, key);
        const int held = next == 0 ? each : __popc(__ballot_sync(0xffffffffu, key == next)), to = min(each, i + held);
        for (int k = i + lane; k < to; k += 32) maxima[threadIdx.x / 32 * each + k] = next;
        if (key == next) key = 0;
        i = to;
    }
}
__device__ __forceinline__ void bound_of(const uint32_t* maxima, int keep, uint32_t& bound) {  // (every thread but one of several equal ones counts)
    const int count = maxima_of(keep) * kWarps;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint32_t mine = maxima[i];
        int place = 0;
#pragma unroll 4
        for (int k = 0; k < count; ++k) place += maxima[k] > mine || (maxima[k] == mine && k < i);
        if (place == keep - 1) bound = mine;
    }
}

struct PartShared {
    uint64_t list[kPartList], best_of[kWarps];
    uint32_t maxima[kWarps * kMostMaxima], bound;
    float tops[kWarps], sums[kWarps], weighted[kWarps];
    float chunk_top[kMostChunks][kThreads];  // a thread's own
    int listed;
};

// The vector of 16 bytes that an end of the row cuts: elements first .. end of it, one by one, and -inf for the others.
template <class T>
__device__ __noinline__ uint4 cut_vector(const T* at, int first, int end) {
    uint4 x = make_uint4(Word<T>::none().bits, Word<T>::none().bits, Word<T>::none().bits, Word<T>::none().bits);
    T e[16 / sizeof(T)];
    __builtin_memcpy(e, &x, 16);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) {
        if (i >= first && i < end) e[i] = at[i];
    }
    __builtin_memcpy(&x, e, 16);
    return x;
}

// Of several holders of (m, sums), all lanes of a warp taking part: the sums relative to `high`, the largest m, of which `first` is one holder.
__device__ __forceinline__ void relative_to(float high, bool first, float m, float& sum, float& weighted) {
    if (first) return;
    const float y = fmaxf((m - high) * kLog2e, kLeast), f = m > kNone ? exp2_approx(y) : 0.0f;
    weighted = (weighted + y * (1.0f + sum)) * f;
    sum = (1.0f + sum) * f;
}

// What a row's alternatives are relative to: the largest logit and log(1 + r).
struct Outcome {
    double top, lse;
    int status;
};

// By one lane: the row's own results.
template <class T>
__device__ __forceinline__ void finish_row(const TokenLogProbsParams& p, Outcome& o, int64_t row, float high, double r, double weighted, int64_t token, float logit) {
    const bool wrong = !(high < -kNone), none = high == kNone, real = token >= 0 && token < p.vocab;
    const double lse = log_of_one_and(r);
    const float nan = __int_as_float(0x7fffffff);
    o.top = high;
    o.lse = lse;
    o.status = wrong ? kRowNonFinite : none ? kRowAllRemoved : p.tokens && !real ? kRowBadToken : kRowOk;
    if (p.tokens) p.log_probs[row] = wrong || none || !real ? nan : (float)(((double)logit - (double)high) - lse);
    if (p.entropy) p.entropy[row] = wrong || none ? nan : (float)(lse - weighted * 0.69314718055994530942 / (1.0 + r));
    if (p.row_status) p.row_status[row] = o.status;
}

__device__ __forceinline__ void put_alternative(const TokenLogProbsParams& p, const Outcome& o, int64_t row, int place, uint64_t key) {
    p.top_log_probs[row * p.top + place] = (float)(((double)from_ordered((uint32_t)(key >> 32)) - o.top) - o.lse);
    p.top_tokens[row * p.top + place] = (int64_t)~(uint32_t)key;
}
__device__ __forceinline__ void put_none(const TokenLogProbsParams& p, int64_t row, int place) {
    p.top_log_probs[row * p.top + place] = kNone;
    p.top_tokens[row * p.top + place] = -1;
}
__device__ __forceinline__ void put_wrong(const TokenLogProbsParams& p, int64_t row, int place) {
    p.top_log_probs[row * p.top + place] = __int_as_float(0x7fffffff);
    p.top_tokens[row * p.top + place] = -1;
}

// The given token of a row and its logit (0 where there is none).
template <class T>
__device__ __forceinline__ float given_logit(const TokenLogProbsParams& p, int64_t row, int64_t& token) {
    token = p.tokens ? p.tokens[row] : 0;
    return p.tokens && token >= 0 && token < p.vocab ? to_float(static_cast<const T*>(p.logits)[row * p.row_stride + token]) : 0.0f;
}

// `whole`: the part is the row.
template <class T, int vectors, bool picks, bool whole>
__device__ __forceinline__ void part_of_row(const TokenLogProbsParams& p, PartShared& s, Outcome& o) {
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
    const int begin = part * p.chunks * kChunk, end = (int)min((int64_t)begin + p.chunks * kChunk, (int64_t)shift + p.vocab);
    const auto column = [&](int chunk, int v) { return begin + chunk * kChunk + (v * kThreads + (int)threadIdx.x) * E; };
    const auto load = [&](int chunk, W (&w)[kWords], bool again) {
#pragma unroll
        for (int v = 0; v < vectors; ++v) {
            const int at = column(chunk, v);
            uint4 x = make_uint4(W::none().bits, W::none().bits, W::none().bits, W::none().bits);
            if (at >= shift && at <= end - E) x = again ? __ldcg(reinterpret_cast<const uint4*>(from + at)) : __ldcs(reinterpret_cast<const uint4*>(from + at));
            else if (at < end && at > shift - E) x = cut_vector(from + at, shift - at, end - at);
            w[4 * v].bits = x.x, w[4 * v + 1].bits = x.y, w[4 * v + 2].bits = x.z, w[4 * v + 3].bits = x.w;
        }
    };

    W best = W::none();  // (the largest so far, of even and of odd places for 16-bit logits)
    float level = kNone;
    float2 sum = {0.0f, 0.0f}, weighted = {0.0f, 0.0f};
    const auto take = [&](int c, W (&x)[kWords]) {
        if constexpr (picks) {
            W high[2] = {x[0], x[1]};
#pragma unroll
            for (int i = 2; i < kWords; ++i) high[i % 2] = high[i % 2].max_with(x[i]);
            const float2 two = high[0].max_with(high[1]).floats();
            s.chunk_top[c][threadIdx.x] = larger(two.x, two.y);
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
        const auto add_up = [&](bool clamp) {
#pragma unroll
            for (int i = 0; i < kWords; i += W::elements == 1 ? 2 : 1) {
                float2 y = x[i].plus(-base);
                if constexpr (W::elements == 1) y.y = x[i + 1].plus(-base).x;
                y = mul_pair(y, make_float2(kLog2e, kLog2e));
                if (clamp) y = make_float2(fmaxf(y.x, kLeast), fmaxf(y.y, kLeast));
                const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                sum = add_pair(sum, e);
                weighted = fma_pair(y, e, weighted);
            }
        };
        // 16-bit logits are brought up to where their weights are 0 in pairs (150 nats below the largest, or a 32nd of that where it is larger, which
        // the type's rounding leaves below 118), but for a largest so low that nothing of the type is.
        const float least = base - fmaxf(150.0f, fabsf(base) * 0x1p-5f);
        if (W::elements == 2 && least > W::lowest) {
            const W floor = W::both(least);
#pragma unroll
            for (int i = 0; i < kWords; ++i) x[i] = x[i].max_with(floor);
            add_up(false);
        } else {
            add_up(true);
        }
    };
    // (Two chunks a turn, one in work and one on its way; unrolled further, the instructions come too late.)
    W w[2][kWords];
    load(0, w[0], false);
#pragma unroll 1
    for (int c = 0; c < p.chunks; c += 2) {
        if (c + 1 < p.chunks) load(c + 1, w[1], false);
        take(c, w[0]);
        if (c + 2 < p.chunks) load(c + 2, w[0], false);
        if (c + 1 < p.chunks) take(c + 1, w[1]);
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
    if (lane == 0) s.tops[warp] = warp_top, s.sums[warp] = own, s.weighted[warp] = own_weighted;
    if constexpr (picks) warp_maxima(top, p.top, s.maxima);
    __syncthreads();
    if constexpr (picks) {
        bound_of(s.maxima, p.top, s.bound);
        __syncthreads();
    }
    if (warp == kWarps - 1) {  // the part's record
        int64_t token = 0;
        float logit = 0.0f;
        if (whole && lane == 0) logit = given_logit<T>(p, row, token);
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
        if (lane == 0) {
            if (whole) finish_row<T>(p, o, row, high, part_sum, part_weighted, token, logit);
            else __stcg(reinterpret_cast<float4*>(p.stats + part_row), make_float4(high, part_sum, part_weighted, 0.0f));
        }
    }
    if constexpr (picks) {
        const int keep = p.top;
        LogProbEntry* entries = p.entries + part_row * keep;
        const auto put = [&](int place, uint64_t key) {
            if constexpr (whole) put_alternative(p, o, row, place, key);
            else __stcg(reinterpret_cast<float2*>(entries + place), make_float2(from_ordered((uint32_t)(key >> 32)), __int_as_float((int)~(uint32_t)key)));
        };
        const float bound = s.bound == 0 ? kNone : from_ordered(s.bound);
        uint32_t hits = 0;  // the chunks that reach the bound; they are read again, out of L2
        for (int c = 0; c < p.chunks; ++c) hits |= (s.chunk_top[c][threadIdx.x] >= bound && s.chunk_top[c][threadIdx.x] > kNone) ? 1u << c : 0u;
        // every logit of those chunks that reaches the bound, with its token
        const auto look = [&](auto use) {
            for (uint32_t rest = hits; rest != 0; rest &= rest - 1) {
                const int c = __ffs(rest) - 1;
                load(c, w[0], true);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const float2 x = w[0][i].floats();
                    const int token = (int)(column(c, i / 4) - shift) + i % 4 * W::elements;
                    if (x.x >= bound && x.x > kNone) use(x.x, token);
                    if constexpr (W::elements == 2) {
                        if (x.y >= bound && x.y > kNone) use(x.y, token + 1);
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
        for (int i = placed + threadIdx.x; i < keep; i += kThreads) {
            if constexpr (whole) put_none(p, row, i);
            else __stcg(reinterpret_cast<float2*>(entries + i), make_float2(kNone, __int_as_float(-1)));
        }
        if (whole && o.status == kRowNonFinite) {
            __syncthreads();
            for (int i = threadIdx.x; i < keep; i += kThreads) put_wrong(p, row, i);
        }
    }
}

struct RowShared {
    uint64_t list[kRowList], best_of[kWarps];
    uint32_t maxima[kWarps * kMostMaxima], bound;
    int listed;
};

// What the parts' blocks have written: out of L2.
__device__ __forceinline__ uint64_t key_of(const LogProbEntry* at) {
    const float2 two = __ldcg(reinterpret_cast<const float2*>(at));
    return two.x > kNone ? entry_key(two.x, __float_as_int(two.y)) : 0;
}

template <class T, bool picks>
__device__ __forceinline__ void whole_row(const TokenLogProbsParams& p, RowShared& s, Outcome& o, int64_t row) {
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
        int64_t token = 0;
        float logit = 0.0f;
        if (lane == 0) logit = given_logit<T>(p, row, token);
        float high = kNone;
        for (int i = lane; i < parts; i += 32) high = larger(high, __ldcg(stats + i).x);
        high = warp_largest(high);
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
        if (lane == 0) finish_row<T>(p, o, row, high, r, weighted, token, logit);
    }
    if constexpr (picks) {
        uint64_t largest = 0;
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) largest = max(largest, held[i]);
        warp_maxima(largest ? from_ordered((uint32_t)(largest >> 32)) : kNone, keep, s.maxima);
        __syncthreads();
        bound_of(s.maxima, keep, s.bound);
        __syncthreads();
        const uint32_t bound = s.bound;
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
        const bool wrong = o.status == kRowNonFinite;
        int placed = wrong ? 0 : min(count, keep);
        const auto put = [&](int place, uint64_t key) { put_alternative(p, o, row, place, key); };
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
            if (wrong) put_wrong(p, row, i);
            else put_none(p, row, i);
        }
    }
}

template <class T, int vectors, bool picks, bool whole>
__global__ void __launch_bounds__(kThreads, kBlocks) token_log_probs_kernel(const __grid_constant__ TokenLogProbsParams p) {
    __shared__ union Shared {
        PartShared part;
        RowShared row;
        __device__ Shared() {}
    } shared;
    __shared__ Outcome outcome;
    __shared__ int is_last;
    part_of_row<T, vectors, picks, whole>(p, shared.part, outcome);
    if constexpr (!whole) {
        const int64_t row = blockIdx.x / (unsigned)p.parts;
        __syncthreads();
        if (threadIdx.x == 0) {  // (release: the block's part, ordered before by the barrier; acquire: the others')
            int before;
            asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + row) : "memory");
            is_last = before == p.parts - 1;
            if (is_last) p.arrived[row] = 0;
        }
        __syncthreads();
        if (is_last) whole_row<T, picks>(p, shared.row, outcome, row);
    }
}

template <class T, int vectors, bool picks>
cudaError_t launch_with(const TokenLogProbsParams& p, cudaStream_t stream) {
    const unsigned blocks = (unsigned)(p.rows * p.parts);
    if (p.parts == 1) token_log_probs_kernel<T, vectors, picks, true><<<blocks, kThreads, 0, stream>>>(p);
    else token_log_probs_kernel<T, vectors, picks, false><<<blocks, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_type(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.vectors == 1) return p.top > 0 ? launch_with<T, 1, true>(p, stream) : launch_with<T, 1, false>(p, stream);
    return p.top > 0 ? launch_with<T, kLongVectors, true>(p, stream) : launch_with<T, kLongVectors, false>(p, stream);
}

}  // namespace

void plan_token_log_probs(TokenLogProbsParams& p, int sm_count) {
    const int E = 16 / element_bytes(p.type);
    // Long parts cost least per logit (what a part costs besides is shared by up to eight chunks); where they would be fewer than the
    // GPU holds at once, shorter ones spread the rows further.
    const auto chunks = [&](int vectors) { return ((int64_t)p.vocab + E - 1 + kThreads * vectors * E - 1) / (kThreads * vectors * E); };
    p.vectors = p.rows * chunks(kLongVectors) < sm_count ? 1 : kLongVectors;
    const int64_t all = chunks(p.vectors);
    // Of the numbers of parts that the chunks allow, the one whose rounds of blocks are done first, a part costing some chunks besides its own.
    constexpr int kBesides = 3;
    int64_t least = 0;
    for (int64_t each = std::min<int64_t>(all, kMostChunks); each > 0; --each) {
        const int64_t parts = (all + each - 1) / each, rounds = (p.rows * parts + sm_count * kBlocks - 1) / (sm_count * kBlocks);
        const int64_t cost = rounds * ((all + parts - 1) / parts + kBesides);
        if (least == 0 || cost < least) least = cost, p.parts = (int)parts;
    }
    p.chunks = (int)((all + p.parts - 1) / p.parts);  // (no part much shorter than the others)
}

cudaError_t launch_token_log_probs(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.type == kFloat32) return launch_type<float>(p, stream);
    if (p.type == kBfloat16) return launch_type<__nv_bfloat16>(p, stream);
    return launch_type<__half>(p, stream);
}

}  // namespace psx
