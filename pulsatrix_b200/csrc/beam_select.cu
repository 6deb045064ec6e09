// Beam search's selection: of all (beam b, token v) of a group, the `keep` with the largest
//
//     value(b, v) = (score_b - log sum_w exp(l_bw)) + l_bv        (double precision; ties: the lowest b, then the lowest v)
//
// First kernel, a block per part of a row (8192 logits, or 2048 where those would leave SMs idle): the logits are read once,
// into registers; the part leaves its maximum, its sum of exponentials and its `keep` best logits in order.  Within a row the
// order by value is the order by logit, so nothing else of the part can be among the group's best.  The `keep` best are found
// without sorting the part: every warp gives the n-th largest of its lanes' maxima, n = ceil(keep / 8), and the smallest of
// those over the eight warps is a bound that at least `keep` logits reach; what reaches it goes on a list (some more than
// `keep`), and an entry's place is the number of keys above its own.  A list that overflows (thousands of equal logits) is
// replaced by `keep` sweeps over the registers.  Bound by HBM: 4 bytes per logit.
//
// Second kernel, a block per group: the rows' normalisers from the parts' sums, then the same selection over the parts' lists.
// It is launched early and waits for the first kernel's end.
//
// The exponentials are summed in float over a thread's 8 or 32 logits, relative to the warp's maximum, and in double from
// there on, in an order that depends on columns alone: equal rows have equal normalisers, so that their candidates tie.
#include "beam_select.cuh"

#include <algorithm>

#include "elements.cuh"

namespace psx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPartList = 1024, kGroupList = 1024;
constexpr int kHeldEntries = 12;  // per thread of the second kernel: 8 beams of 19 parts with 16 each in all
constexpr float kNone = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

// Floats as integers of the same order (NaN aside); 0 is below every number.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }

// -0 and +0 are equal: both as +0.
__device__ __forceinline__ uint64_t entry_key(float logit, int token) {
    return (uint64_t)ordered(logit + 0.0f) << 32 | (uint32_t)~token;
}

// A number that at least `keep` of the block's numbers reach, given every thread's largest (-inf where it has none): see
// above.  Lanes of equal maxima leave together, which can only lower it.
__device__ __forceinline__ uint32_t warp_bound(float largest, int keep, uint32_t* top) {
    uint32_t key = ordered(largest), bound = 0;
    for (int n = (keep + kWarps - 1) / kWarps; n > 0; --n) {
        bound = __reduce_max_sync(0xffffffffu, key);
        if (top) *top = bound, top = nullptr;
        key = key == bound ? 0u : key;
        if (bound <= ordered(kNone)) return 0;
    }
    return bound;
}

__device__ __forceinline__ uint64_t block_max(uint64_t key, uint64_t* shared) {
    for (int step = 16; step > 0; step /= 2) key = max(key, __shfl_xor_sync(0xffffffffu, key, step));
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = key;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) key = max(key, shared[w]);
    __syncthreads();
    return key;
}

template <int values, bool aligned>
__global__ void __launch_bounds__(kThreads) beam_parts_kernel(const __grid_constant__ BeamSelectParams p) {
    constexpr int kPart = kThreads * values;
    __shared__ uint64_t list[kPartList], best_of[kWarps];
    __shared__ uint32_t bounds[kWarps], tops[kWarps];
    __shared__ double sums[kWarps];
    __shared__ int listed, not_finite;
    const int64_t part_row = blockIdx.x;
    const int64_t row = part_row / p.parts;
    const int part = (int)(part_row % p.parts), keep = p.keep, first = part * kPart;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    BeamEntry* entries = p.entries + part_row * keep;
    const float score = p.scores[row];
    const bool ended = p.finished && p.finished[row];
    if (ended || score == kNone) {  // nothing of this row is read
        for (int i = threadIdx.x; i < keep; i += kThreads) {
            const bool offers = ended && part == 0 && i == 0;
            entries[i] = {offers ? 0.0f : kNone, offers ? (int)p.finished_token : -1};
        }
        if (threadIdx.x == 0) p.part_stats[part_row] = {0.0, kNone, 0};
        asm volatile("griddepcontrol.launch_dependents;");
        return;
    }
    if (threadIdx.x == 0) listed = 0, not_finite = 0;

    float v[values];
    const float* from = p.logits + row * p.row_stride;
    // Column of a thread's j-th logit: fours of neighbours where the rows are aligned, neighbours on neighbouring lanes else.
    const auto column = [&](int j) {
        return aligned ? first + j / 4 * (kThreads * 4) + (int)threadIdx.x * 4 + j % 4 : first + j * kThreads + (int)threadIdx.x;
    };
    if constexpr (aligned) {
#pragma unroll
        for (int j = 0; j < values; j += 4) {
            float4 x = make_float4(kNone, kNone, kNone, kNone);
            if (column(j) < p.vocab) x = __ldcs(reinterpret_cast<const float4*>(from + column(j)));
            v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < values; ++j) v[j] = column(j) < p.vocab ? __ldcs(from + column(j)) : kNone;
    }
    float largest = kNone;
    bool wrong = false;
#pragma unroll
    for (int j = 0; j < values; ++j) {
        largest = fmaxf(largest, v[j]);
        wrong |= !(v[j] < -kNone);
    }
    uint32_t top_key;
    const uint32_t mine = warp_bound(largest, keep, &top_key);
    const float top = from_ordered(top_key);
    float sum = 0.0f;
    if (top > kNone) {
#pragma unroll
        for (int j = 0; j < values; ++j) sum += exp2_approx((v[j] - top) * kLog2e);
    }
    double total = sum;
#pragma unroll
    for (int step = 16; step > 0; step /= 2) total += __shfl_xor_sync(0xffffffffu, total, step);
    if (lane == 0) {
        bounds[warp] = mine;
        tops[warp] = top_key;
        sums[warp] = total;
    }
    const bool any_wrong = __any_sync(0xffffffffu, wrong);
    __syncthreads();
    if (any_wrong && lane == 0) not_finite = 1;
    uint32_t bound_key = bounds[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound_key = min(bound_key, bounds[w]);
    const float bound = bound_key == 0 ? kNone : from_ordered(bound_key);
    if (largest >= bound && largest > kNone) {
#pragma unroll
        for (int j = 0; j < values; ++j) {
            if (v[j] >= bound && v[j] > kNone) {
                const int at = atomicAdd(&listed, 1);
                if (at < kPartList) list[at] = entry_key(v[j], column(j));
            }
        }
    }
    __syncthreads();
    const int count = listed;
    if (threadIdx.x < 32) {  // the part's record
        const float warp_top = lane < kWarps ? from_ordered(tops[lane]) : kNone;
        float part_top = warp_top;
        for (int step = 16; step > 0; step /= 2) part_top = fmaxf(part_top, __shfl_xor_sync(0xffffffffu, part_top, step));
        double part_sum = lane < kWarps && warp_top > kNone ? sums[lane] * exp((double)warp_top - (double)part_top) : 0.0;
        for (int step = 16; step > 0; step /= 2) part_sum += __shfl_xor_sync(0xffffffffu, part_sum, step);
        if (lane == 0) p.part_stats[part_row] = {part_sum, part_top, not_finite};
    }
    int placed = min(count, keep);
    if (count <= kPartList) {
        for (int e = threadIdx.x; e < count; e += kThreads) {
            const uint64_t key = list[e];
            int place = 0;
            for (int k = 0; k < count; ++k) place += list[k] > key;
            if (place < keep) entries[place] = {from_ordered((uint32_t)(key >> 32)), (int)~(uint32_t)key};
        }
    } else {
        uint64_t last = ~0ull;
        for (placed = 0; placed < keep; ++placed) {
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < values; ++j) {
                const uint64_t key = v[j] > kNone ? entry_key(v[j], column(j)) : 0;
                if (key < last) best = max(best, key);
            }
            best = block_max(best, best_of);
            if (best == 0) break;
            if (threadIdx.x == 0) entries[placed] = {from_ordered((uint32_t)(best >> 32)), (int)~(uint32_t)best};
            last = best;
        }
    }
    for (int i = placed + threadIdx.x; i < keep; i += kThreads) entries[i] = {kNone, -1};
    asm volatile("griddepcontrol.launch_dependents;");
}

struct Candidate {
    double value;
    uint64_t place;  // beam << 32 | token
};

__device__ __forceinline__ bool ahead(const Candidate& a, const Candidate& b) {
    return a.value > b.value || (a.value == b.value && a.place < b.place);
}

// The value as a float, in an order that rounding keeps; what is below the lowest float counts as that, so that it stays a candidate.
__device__ __forceinline__ float as_float(double value) { return value > (double)kNone ? fmaxf((float)value, -3.402823466e38f) : kNone; }

__global__ void __launch_bounds__(kThreads) beam_groups_kernel(const __grid_constant__ BeamSelectParams p) {
    __shared__ double base[kMostSelectBeams];  // score - normaliser; -inf: the beam offers nothing
    __shared__ Candidate list[kGroupList], best_of[kWarps];
    __shared__ uint32_t bounds[kWarps];
    __shared__ int listed, not_finite;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t group = blockIdx.x;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, keep = p.keep;
    if (threadIdx.x == 0) listed = 0, not_finite = 0;
    // The first entries of every thread are asked for ahead of the normalisers, and kept.
    const BeamEntry* entries = p.entries + group * p.beams * p.parts * keep;
    const int per_beam = p.parts * keep, all = p.beams * per_beam;
    BeamEntry held[kHeldEntries];
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        const int e = i * kThreads + threadIdx.x;
        held[i] = e < all ? entries[e] : BeamEntry{kNone, -1};
    }
    __syncthreads();
    for (int b = warp; b < p.beams; b += kWarps) {
        const int64_t row = group * p.beams + b;
        const BeamPart* parts = p.part_stats + row * p.parts;
        const float score = p.scores[row];
        const bool ended = p.finished && p.finished[row];
        float top = kNone;
        int wrong = !(score < -kNone);
        for (int i = lane; i < p.parts; i += 32) {
            const BeamPart part = parts[i];
            top = fmaxf(top, part.top);
            wrong |= part.not_finite;
        }
        for (int step = 16; step > 0; step /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
        double sum = 0.0;
        for (int i = lane; i < p.parts; i += 32) {
            const BeamPart part = parts[i];
            if (part.top > kNone) sum += part.sum * exp((double)part.top - (double)top);
        }
        for (int step = 16; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
        wrong = __any_sync(0xffffffffu, wrong);
        if (lane == 0) {
            if (wrong) not_finite = 1;
            base[b] = ended ? (double)score : sum > 0.0 ? (double)score - ((double)top + log(sum)) : (double)kNone;
        }
    }
    __syncthreads();
    const auto candidate_of = [&](int e, BeamEntry entry) {
        const int b = e / per_beam;
        return Candidate{base[b] + (double)entry.logit, (uint64_t)b << 32 | (uint32_t)entry.token};
    };
    const auto candidate = [&](int e) { return candidate_of(e, entries[e]); };
    constexpr int kHeld = kHeldEntries * kThreads;
    float largest = kNone;
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        const int e = i * kThreads + threadIdx.x;
        if (e < all) largest = fmaxf(largest, as_float(candidate_of(e, held[i]).value));
    }
#pragma unroll 4
    for (int e = kHeld + threadIdx.x; e < all; e += kThreads) largest = fmaxf(largest, as_float(candidate(e).value));
    const uint32_t mine = warp_bound(largest, keep, nullptr);
    if (lane == 0) bounds[warp] = mine;
    __syncthreads();
    uint32_t bound_key = bounds[0];
    for (int w = 1; w < kWarps; ++w) bound_key = min(bound_key, bounds[w]);
    const float bound = bound_key == 0 ? kNone : from_ordered(bound_key);
    // (rounding to float keeps the order: what is at or above the bound in double is so in float)
    if (largest >= bound && largest > kNone) {
        const auto offer = [&](const Candidate& c) {
            if (c.value > (double)kNone && as_float(c.value) >= bound) {
                const int at = atomicAdd(&listed, 1);
                if (at < kGroupList) list[at] = c;
            }
        };
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) {
            const int e = i * kThreads + threadIdx.x;
            if (e < all) offer(candidate_of(e, held[i]));
        }
        for (int e = kHeld + threadIdx.x; e < all; e += kThreads) offer(candidate(e));
    }
    __syncthreads();
    const int count = listed;
    const bool wrong = not_finite != 0;
    int placed = wrong ? 0 : min(count, keep);
    const auto put = [&](int place, const Candidate& c) {
        const int64_t at = group * keep + place;
        p.out_scores[at] = as_float(c.value);
        p.parents[at] = (int64_t)(c.place >> 32);
        p.tokens[at] = (int64_t)(uint32_t)c.place;
    };
    if (wrong) {
    } else if (count <= kGroupList) {
        for (int e = threadIdx.x; e < count; e += kThreads) {
            const Candidate c = list[e];
            int place = 0;
            for (int k = 0; k < count; ++k) place += ahead(list[k], c);
            if (place < keep) put(place, c);
        }
    } else {  // more that tie at the bound than the list holds: sweep after sweep, the best that is behind the last one
        Candidate last{(double)-kNone, 0};
        for (placed = 0; placed < keep; ++placed) {
            Candidate best{(double)kNone, ~0ull};
            for (int e = threadIdx.x; e < all; e += kThreads) {
                const Candidate c = candidate(e);
                if (ahead(last, c) && ahead(c, best)) best = c;
            }
            for (int step = 16; step > 0; step /= 2) {
                const Candidate other{__shfl_xor_sync(0xffffffffu, best.value, step), __shfl_xor_sync(0xffffffffu, best.place, step)};
                if (ahead(other, best)) best = other;
            }
            if (lane == 0) best_of[warp] = best;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w) {
                if (ahead(best_of[w], best)) best = best_of[w];
            }
            __syncthreads();
            if (best.value == (double)kNone) break;
            if (threadIdx.x == 0) put(placed, best);
            last = best;
        }
    }
    for (int i = placed + threadIdx.x; i < keep; i += kThreads) {
        p.out_scores[group * keep + i] = kNone;
        p.parents[group * keep + i] = -1;
        p.tokens[group * keep + i] = -1;
    }
    if (threadIdx.x == 0 && p.group_status) p.group_status[group] = wrong ? 4 : placed == 0 ? 5 : 0;  // (psx_row_status)
}

}  // namespace

void plan_beam_select(BeamSelectParams& p, int sm_count) {
    const int64_t rows = p.groups * p.beams;
    // 32 logits per thread keep enough loads in flight; with fewer blocks than SMs the shorter parts spread the row further.
    p.values = rows * ((p.vocab + kThreads * 32 - 1) / (kThreads * 32)) < sm_count ? 8 : 32;
    p.parts = (p.vocab + kThreads * p.values - 1) / (kThreads * p.values);
    p.aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.row_stride % 4 == 0 && p.vocab % 4 == 0;
}

cudaError_t launch_beam_select(const BeamSelectParams& p, cudaStream_t stream) {
    const unsigned blocks = (unsigned)(p.groups * p.beams * p.parts);
    if (p.values == 8) {
        if (p.aligned) beam_parts_kernel<8, true><<<blocks, kThreads, 0, stream>>>(p);
        else beam_parts_kernel<8, false><<<blocks, kThreads, 0, stream>>>(p);
    } else {
        if (p.aligned) beam_parts_kernel<32, true><<<blocks, kThreads, 0, stream>>>(p);
        else beam_parts_kernel<32, false><<<blocks, kThreads, 0, stream>>>(p);
    }
    if (const cudaError_t e = cudaGetLastError()) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)p.groups);
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, beam_groups_kernel, p);
}

}  // namespace psx
