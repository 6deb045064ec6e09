// Log-probabilities of given tokens, with the entropy of the row and its largest alternatives, in one pass over the logits.
//
// With m the row's largest logit and sums over all logits but one that is m,
//     r = sum exp(x - m),   log p(t) = (x_t - m) - log(1 + r),   H = log(1 + r) + sum (m - x) exp(x - m) / (1 + r).
// The largest itself stays out of the sums, so that a row whose token is nearly certain has the digits of r = 1e-9 and not those of 1 + r: a
// thread keeps the largest of its logits aside, and whatever is not larger than it (or the one that it replaces) joins the sums, relative to
// the thread's largest so far.  16-bit logits are compared in pairs as they come.
//
// The row is cut into 1 to 16 parts, the CTAs of a cluster; a thread takes up to four vectors of 16 bytes at a time, with the next ones on their way (two
// instead of four: 220 us instead of 120 for 2048 rows of 151,936 bf16 logits).  The `top` best are found by a bound that at least `top` logits reach: each
// part's is the top-th largest of its threads' largest, the row's the largest of those, or the smallest of what each part's share of them reaches.
// A thread whose largest of some chunks reaches it looks at them again, out of L2, and puts what reaches the bound on its CTA's list; the first CTA brings the
// lists together, and an entry's place is the number of keys above its own.  A list that overflows (thousands of equal logits) is replaced by `top` sweeps.
// Records, bounds and lists go through the cluster's shared memory: there is no scratch and nothing to be zero before a call.  (Lists and records in global
// memory, joined by the part that ends last: 64 rows of 8000 logits, 20 alternatives, 12.4 us instead of 8.3.)
//
// Rows need not be aligned: vectors are those of memory, and where one is cut by an end of the row its elements are read one by one.  Bound by HBM, the
// logits once, and nearly so by instructions for 16-bit logits, 9.0 for each: 2048 rows of 151,936 bf16 logits take 120 us when replayed (5.2 TB/s, issue slots 58 % busy;
// 107 without alternatives; 124 to 133, by the machine, on other logits every time), 1000 of 128,256 fp32 logits 93 (5.5 TB/s).
#include "token_log_probs.cuh"

#include <algorithm>
#include <type_traits>

#include "once_per_device.hpp"
#include "psx_device.cuh"
#include "row_selection.cuh"

namespace psx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostGroups = 32;  // of a part's chunks
constexpr int kLongVectors = 4;
constexpr int kBlocks = 4;  // that an SM holds
// Chunks of one vector that a part has at most, and where rows come in several rounds of an SM's CTAs: there more are slower than a quarter as many of four vectors,
// whatever their chains (in us, with chunks of one vector and of four: 600 rows of 12,000 fp32 logits, twelve chunks, 14.4 and 16.5; 2000 rows of 8000, eight, 26.8 and
// 28.1, of 12,000, twelve, 37 and 33; 8000 rows of 16,000 164 and 132, of 50,257 453 and 271; 8000 of 32,000 bf16 logits, sixteen, 191 and 169, of 151,936 815 and 433).
constexpr int kMostShort = 32, kMostShortInRounds = 8;
// Chunks whose sums a thread holds as floats: of 294,912 logits, so that the vocabularies of today have no use for more (handing on costs 2 to 4 % of a row's time).
template <class T>
constexpr int kHandOn = 18 * sizeof(T);
constexpr int kMostMaxima = (kMostTop + kWarps - 1) / kWarps + 2;  // of a warp
constexpr int kList = 1024;
constexpr int kMostParts = 16;  // of a row: a cluster's CTAs
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
// `share`: the same for its `share_of`-th largest.
__device__ __forceinline__ void bound_of(const uint32_t* maxima, int keep, int share_of, uint32_t& bound, uint32_t& share) {
    const int count = maxima_of(keep) * kWarps;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint32_t mine = maxima[i];
        int place = 0;
#pragma unroll 4
        for (int k = 0; k < count; ++k) place += maxima[k] > mine || (maxima[k] == mine && k < i);
        if (place == keep - 1) bound = mine;
        if (place == share_of - 1) share = mine;
    }
}

// What a row's alternatives are relative to: the largest logit and log(1 + r).
struct Outcome {
    double top, lse;
    int status;
};

// A thread's sums of all chunks but the last few, relative to `level`.
struct Held {
    double sum[kThreads], weighted[kThreads];
    float level[kThreads];
};

struct Shared {
    union {
        alignas(16) uint64_t list[kList];  // what reaches the bound
        Held held;                         // before there is a list
    };
    uint64_t best_of[kWarps], best[2];
    float4 record;         // the part's largest logit and its two sums
    Outcome outcome;       // the first part's, and the given token and its logit
    int64_t token;
    float given;
    uint32_t maxima[kWarps * kMostMaxima], bound, share;
    float tops[kWarps], sums[kWarps], weighted[kWarps];
    alignas(16) float group_top[kMostGroups][kThreads];  // a thread's own
    uint32_t listed, together;
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

// A thread's sums of some chunks, relative to `level`, go to those that it holds in double precision.
__device__ __noinline__ void hand_on(Held& held, float level, float sum, float weighted) {
    const int i = threadIdx.x;
    const double less = fmax(((double)held.level[i] - (double)level) * 1.4426950408889634, -2000.0), factor = exp2(less);  // (2^-2000 is 0)
    held.weighted[i] = (held.weighted[i] + less * held.sum[i]) * factor + (double)weighted;
    held.sum[i] = held.sum[i] * factor + (double)sum;
    held.level[i] = level;
}

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

// The given token of a row and its logit (0 where there is none).
template <class T>
__device__ __forceinline__ float given_logit(const TokenLogProbsParams& p, int64_t row, int64_t& token) {
    token = p.tokens ? p.tokens[row] : 0;
    return p.tokens && token >= 0 && token < p.vocab ? to_float(static_cast<const T*>(p.logits)[row * p.row_stride + token]) : 0.0f;
}

// ---- the cluster's shared memory --------------------------------------------------------------------------------------------
// `alone`: a cluster of one CTA.  All threads of the CTAs meet, each by itself.
template <bool alone>
struct Cluster {
    __device__ __forceinline__ static void meets() {
        if constexpr (alone) __syncthreads();
        else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }
    // Where CTA `rank` has what this CTA has at p.
    __device__ __forceinline__ static uint32_t at(const void* p, int rank) {
        const uint32_t here = (uint32_t)__cvta_generic_to_shared(p);
        if constexpr (alone) return here;
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
        return there;
    }
    __device__ __forceinline__ static uint32_t load_u32(uint32_t at) {
        uint32_t x;
        if constexpr (alone) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
        else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
        return x;
    }
    __device__ __forceinline__ static uint64_t load_u64(uint32_t at) {
        uint64_t x;
        if constexpr (alone) asm volatile("ld.shared.u64 %0, [%1];" : "=l"(x) : "r"(at) : "memory");
        else asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(at) : "memory");
        return x;
    }
    __device__ __forceinline__ static float4 load_f4(uint32_t at) {
        float4 x;
        if constexpr (alone) asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
        else asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
        return x;
    }
};

// `many`: a part has more than kHandOn<T> chunks.
template <class T, int vectors, bool picks, bool alone, bool many>
__global__ void __launch_bounds__(kThreads, kBlocks) token_log_probs_kernel(const __grid_constant__ TokenLogProbsParams p) {
    constexpr int E = 16 / sizeof(T), kChunk = kThreads * vectors * E, kWords = vectors * 4;
    using W = Word<T>;
    using C = Cluster<alone>;
    __shared__ Shared s;
    const int parts = alone ? 1 : p.parts;
    const int64_t row = blockIdx.x / (unsigned)parts;
    const int part = alone ? 0 : (int)(blockIdx.x % (unsigned)parts), warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    grid_dependency_wait();
    grid_dependents_may_launch();
    if (threadIdx.x == 0) s.listed = 0, s.together = 0;
    // Elements are counted from the 16-byte boundary that is not behind the row's first one.
    const T* from = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int shift = (int)(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
    from -= shift;
    const int begin = part * p.chunks * kChunk, end = (int)min((int64_t)begin + p.chunks * kChunk, (int64_t)shift + p.vocab);
    const auto column = [&](int chunk, int v) { return begin + chunk * kChunk + (v * kThreads + (int)threadIdx.x) * E; };
    const auto load = [&](int chunk, W (&w)[kWords]) {
#pragma unroll
        for (int v = 0; v < vectors; ++v) {
            const int at = column(chunk, v);
            uint4 x = make_uint4(W::none().bits, W::none().bits, W::none().bits, W::none().bits);
            if (at >= shift && at <= end - E) x = __ldcg(reinterpret_cast<const uint4*>(from + at));
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
            const float chunk_top = larger(two.x, two.y);
            if (p.group == 1) {
                s.group_top[c][threadIdx.x] = chunk_top;
            } else {
                float& held = s.group_top[c / p.group][threadIdx.x];
                held = c % p.group == 0 ? chunk_top : larger(held, chunk_top);
            }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {  // the larger one is kept aside
            const W lower = best.min_with(x[i]);
            best = best.max_with(x[i]);
            x[i] = lower;
        }
        const float2 two = best.floats();
        // (Behind logits of -inf alone the lowest number, so that the factor of the empty sums is never above 1: 0 would make it infinite before a first logit of -89.)
        const float base = fmaxf(fmaxf(two.x, two.y), -0x1.fffffep127f);
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
    // Sums of floats lose a unit with every addition and two with every new largest: in rows of many chunks they go to sums in double precision time after time.
    if constexpr (many) s.held.sum[threadIdx.x] = s.held.weighted[threadIdx.x] = 0.0, s.held.level[threadIdx.x] = kNone;
    // (Two chunks a turn, one in work and one on its way; unrolled further, the instructions come too late.)
    W w[2][kWords];
    load(0, w[0]);
    if (part == 0 && threadIdx.x == 0) {  // (here its two trips to memory are nobody's)
        int64_t token;
        s.given = given_logit<T>(p, row, token);
        s.token = token;
    }
#pragma unroll 1
    for (int c = 0; c < p.chunks; c += 2) {
        if (c + 1 < p.chunks) load(c + 1, w[1]);
        take(c, w[0]);
        if (c + 2 < p.chunks) load(c + 2, w[0]);
        if (c + 1 < p.chunks) take(c + 1, w[1]);
        if constexpr (many) {
            if ((c + 2) % kHandOn<T> == 0) {
                hand_on(s.held, level, sum.x + sum.y, weighted.x + weighted.y);
                sum = weighted = make_float2(0.0f, 0.0f);
            }
        }
    }
    // The thread's own: the smaller of the two that are aside joins the sums.
    const float2 aside = best.floats();
    const float top = larger(aside.x, aside.y);
    float own = sum.x + sum.y, own_weighted = weighted.x + weighted.y;
    if constexpr (many) {
        hand_on(s.held, level, own, own_weighted);
        own = (float)s.held.sum[threadIdx.x], own_weighted = (float)s.held.weighted[threadIdx.x];
    }
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
        bound_of(s.maxima, p.top, (p.top + parts - 1) / parts, s.bound, s.share);
        __syncthreads();
    }
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
        if (lane == 0) s.record = make_float4(high, part_sum, part_weighted, 0.0f);
    }
    float bound = kNone;
    uint32_t hits = 0;  // the groups of chunks that reach it; they are read again, out of L2
    const auto look_from = [&](uint32_t key) {
        bound = key == 0 ? kNone : from_ordered(key);
        const int groups = (p.chunks + p.group - 1) / p.group;
        hits = 0;
        for (int g = 0; g < groups; ++g) hits |= (s.group_top[g][threadIdx.x] >= bound && s.group_top[g][threadIdx.x] > kNone) ? 1u << g : 0u;
    };
    // every logit of those that reaches the bound, with its token
    const auto look = [&](auto use) {
        for (uint32_t rest = hits; rest != 0; rest &= rest - 1) {
            const int g = __ffs(rest) - 1, last = min((g + 1) * p.group, p.chunks);
            for (int c = g * p.group; c < last; ++c) {
                load(c, w[0]);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const float2 x = w[0][i].floats();
                    const int token = column(c, i / 4) - shift + i % 4 * W::elements;
                    if (x.x >= bound && x.x > kNone) use(x.x, token);
                    if constexpr (W::elements == 2) {
                        if (x.y >= bound && x.y > kNone) use(x.y, token + 1);
                    }
                }
            }
        }
    };
    if constexpr (picks) {
        look_from(s.bound);
        look([&](float x, int token) {
            const uint32_t at = atomicAdd(&s.listed, 1u);
            if (at < kList) s.list[at] = entry_key(x, token);
        });
    }
    C::meets();
    if (part == 0 && warp == 0) {  // the row's
        const float4 x = lane < parts ? C::load_f4(C::at(&s.record, lane)) : make_float4(kNone, 0.0f, 0.0f, 0.0f);
        const float high = warp_largest(x.x);
        const unsigned holds = __ballot_sync(0xffffffffu, lane < parts && x.x == high);
        float sum = x.y, w = x.z;
        relative_to(high, lane == __ffs(holds) - 1, x.x, sum, w);
        double r = sum, all_weighted = w;
#pragma unroll
        for (int step = kMostParts / 2; step > 0; step /= 2) {
            r += __shfl_xor_sync(0xffffffffu, r, step);
            all_weighted += __shfl_xor_sync(0xffffffffu, all_weighted, step);
        }
        if (lane == 0) finish_row<T>(p, s.outcome, row, high, r, all_weighted, s.token, s.given);
    }
    if constexpr (!picks) {
        if (!alone) C::meets();  // (the records are read until then)
        return;
    }

    // What the parts have listed, and the row's bound: at least `top` logits reach the largest of theirs; and, each part giving its share of them, the
    // smallest of those.
    const int listed = lane < parts ? (int)C::load_u32(C::at(&s.listed, lane)) : 0;
    const uint32_t reached = __reduce_max_sync(0xffffffffu, lane < parts ? C::load_u32(C::at(&s.bound, lane)) : 0u);
    const uint32_t shared_out = __reduce_min_sync(0xffffffffu, lane < parts ? C::load_u32(C::at(&s.share, lane)) : 0xffffffffu);
    const uint32_t bound_key = max(reached, shared_out);
    const int keep = p.top;
    int placed;
    if (!__any_sync(0xffffffffu, listed > kList) && (int)__reduce_add_sync(0xffffffffu, (unsigned)listed) <= 2 * kList) {  // (the same in all warps)
        if (part == 0) {
            const uint64_t* list = s.list;
            int count = listed;
            if constexpr (alone) {
                count = __shfl_sync(0xffffffffu, listed, 0);
                __syncthreads();  // (the row's outcome)
            } else {  // the first CTA brings them together, where its threads kept their groups', which are done with
                uint64_t* together = reinterpret_cast<uint64_t*>(s.group_top);
                for (int i = warp; i < parts; i += kWarps) {
                    const int of_part = __shfl_sync(0xffffffffu, listed, i);
                    for (int e = lane; e < of_part; e += 32) {
                        const uint64_t key = C::load_u64(C::at(&s.list[e], i));
                        if ((uint32_t)(key >> 32) >= bound_key) together[atomicAdd(&s.together, 1u)] = key;
                    }
                }
                __syncthreads();
                list = together;
                count = (int)s.together;
            }
            const bool wrong = s.outcome.status == kRowNonFinite;
            for (int e = threadIdx.x; e < (wrong ? 0 : count); e += kThreads) {
                const uint64_t key = list[e];
                int place = 0;
#pragma unroll 4
                for (int k = 0; k < count / 2; ++k) {
                    const ulonglong2 two = reinterpret_cast<const ulonglong2*>(list)[k];
                    place += (two.x > key) + (two.y > key);
                }
                if (count % 2) place += list[count - 1] > key;
                if (place < keep) put_alternative(p, s.outcome, row, place, key);
            }
            placed = min(count, keep);
        }
    } else {  // thousands that tie at the bound: sweep after sweep, the best that is behind the last one
        look_from(bound_key);
        uint64_t last = ~0ull;
        for (placed = 0; placed < keep; ++placed) {
            uint64_t next = 0;
            look([&](float x, int token) {
                const uint64_t key = entry_key(x, token);
                if (key < last) next = max(next, key);
            });
            next = block_max<kWarps>(next, s.best_of);
            uint64_t& mine = s.best[placed % 2];  // (two that take turns: one meeting a sweep is enough)
            if (threadIdx.x == 0) mine = next;
            C::meets();
            for (int i = 0; i < parts; ++i) next = max(next, C::load_u64(C::at(&mine, i)));
            if (next == 0) break;
            if (part == 0 && threadIdx.x == 0) put_alternative(p, s.outcome, row, placed, next);
            last = next;
        }
    }
    if (part == 0) {
        const bool wrong = s.outcome.status == kRowNonFinite;
        if (wrong) __syncthreads();  // (what the sweeps have put is put over)
        for (int i = (wrong ? 0 : placed) + threadIdx.x; i < keep; i += kThreads) {
            p.top_log_probs[row * keep + i] = wrong ? __int_as_float(0x7fffffff) : kNone;
            p.top_tokens[row * keep + i] = -1;
        }
    }
    if (!alone) C::meets();  // (records, lists and the sweeps' best are read until then)
}

template <class T, int vectors, bool picks, bool many>
cudaError_t launch_with(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.parts == 1) {
        return launch_overlapping(token_log_probs_kernel<T, vectors, picks, true, many>, dim3((unsigned)p.rows), dim3(kThreads), 0, stream, p);
    }
    const auto kernel = token_log_probs_kernel<T, vectors, picks, false, many>;
    if (p.parts > 8) {  // (more than any device must hold)
        static OncePerDevice raised;
        int device = 0;
        if (const cudaError_t e = cudaGetDevice(&device)) return e;
        const cudaError_t e = raised.run(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
        if (e != cudaSuccess) return e;
    }
    return launch_overlapping(kernel, dim3((unsigned)(p.rows * p.parts)), dim3(kThreads), 0, stream, p, (unsigned)p.parts);
}

template <class T>
cudaError_t launch_type(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.vectors == 1) return p.top > 0 ? launch_with<T, 1, true, false>(p, stream) : launch_with<T, 1, false, false>(p, stream);
    if (p.chunks > kHandOn<T>) return p.top > 0 ? launch_with<T, kLongVectors, true, true>(p, stream) : launch_with<T, kLongVectors, false, true>(p, stream);
    return p.top > 0 ? launch_with<T, kLongVectors, true, false>(p, stream) : launch_with<T, kLongVectors, false, false>(p, stream);
}

}  // namespace

void plan_token_log_probs(TokenLogProbsParams& p, int sm_count) {
    const int E = 16 / element_bytes(p.type);
    // The cluster size and the vectors of a chunk that a row takes least time with.  In us, as measured with 8 alternatives: one CTA by itself takes `chain`
    // for its steps and `chunk` for each of its chunks, which come one behind the other; every further one on its SM adds what its instructions and
    // bytes take there.  (64 x 151,936 bf16 in 1, 2, 4, 8, 16 parts: 21.2, 15.5, 13.2, 14.2, 27.5; 2000 x 4000 in one: 23.1 with one vector, 28.7 with
    // four; 700 x 128,256 fp32 in 1, 2, 4: 84, 79, 91.)  Clusters of 16 are for few rows: they leave SMs idle where there are many.
    double least = 0.0;
    for (const int vectors : {kLongVectors, 1}) {
        const double chunk = vectors == 1 ? 0.375 : 0.79, chain = vectors == 1 ? 4.3 : 5.2, further = vectors == 1 ? 1.2 : 1.7, further_chunk = 0.09 * vectors;
        const int64_t elements = kThreads * vectors * E, all = (p.vocab + E - 1 + elements - 1) / elements;
        for (int parts = 1; parts <= kMostParts; parts *= 2) {
            const int64_t each = (all + parts - 1) / parts;
            const double beside = std::max(1.0, (double)(p.rows * parts) / sm_count);
            if (vectors == 1 && each > (beside > 2.0 * kBlocks ? kMostShortInRounds : kMostShort)) continue;
            if (parts > 1 && (each * (parts - 1) >= all || (parts == kMostParts && beside > 1.0))) continue;  // (a part would be empty)
            const double cost = each * chunk + chain + (parts > 1 ? 1.0 : 0.0) + (beside - 1.0) * (further + further_chunk * each);
            if (least == 0.0 || cost < least) least = cost, p.parts = parts, p.vectors = vectors, p.chunks = (int)each;
        }
    }
    p.group = (p.chunks + kMostGroups - 1) / kMostGroups;
}

cudaError_t launch_token_log_probs(const TokenLogProbsParams& p, cudaStream_t stream) {
    if (p.type == kFloat32) return launch_type<float>(p, stream);
    if (p.type == kBfloat16) return launch_type<__nv_bfloat16>(p, stream);
    return launch_type<__half>(p, stream);
}

}  // namespace psx
