// Beam search's selection: of all (beam b, token v) of a group, the `keep` with the largest
//
//     value(b, v) = (score_b - log sum_w exp(l_bw)) + l_bv        (added in double; ties: the lowest b, then the lowest v)
//
// A block takes a part of a row: the logits are read once, in chunks of 16 per thread (4 where that would leave SMs
// idle) with the next chunk on its way, a running maximum and sum per thread; the part leaves its maximum, its sum of
// exponentials and its `keep` best logits in order.  Within a row the order by value is the order by logit, so nothing else of
// the part can be among the group's best.  The `keep` best are found without sorting the part: every warp gives the n-th
// largest of its lanes' maxima, n = ceil(keep / 8), and the smallest of those over the eight warps is a bound that at least
// `keep` logits reach.  The few chunks whose maximum reaches it are read again, out of L2, and what reaches it goes on a list
// (some more than `keep`); an entry's place is the number of keys above its own.  A list that overflows (thousands of equal
// logits) is replaced by `keep` sweeps over those chunks.  Bound by HBM: 4 bytes per logit.
//
// The block of a group that ends last goes on with the group: the rows' normalisers from the parts' sums, then the same selection over
// the parts' lists.  (A second kernel for that cost one call of 4 beams 3 us on the GPU and as much on the host.)
//
// The exponentials are summed in float over a thread's logits, relative to its maximum so far, and in double from there on, in
// an order that depends on columns alone: equal rows have equal normalisers, so that their candidates tie.  In units of 2^-24 of the sum: 1.1 for
// a term's exponent, 4 for its exponential, 5 for a chunk of 16 in four sums, 8 for a thread's running sum, 6 each for at most seven factors of a
// new maximum and three in the joins: less than 80, 4.8e-6 of the logarithm.
#include "beam_select.cuh"

#include <algorithm>

#include "row_selection.cuh"

namespace psx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostChunks = 8;  // of a part
constexpr int kPartList = 1024, kGroupList = 1024;
constexpr int kHeldEntries = 8;  // per thread, of the parts' lists

struct PartShared {
    uint64_t list[kPartList], best_of[kWarps];
    uint32_t bounds[kWarps], tops[kWarps];
    double sums[kWarps];
    int listed;
};

template <int values, bool aligned>
__device__ __forceinline__ void part_of_row(const BeamSelectParams& p, PartShared& s) {
    constexpr int kChunk = kThreads * values;
    const int64_t part_row = blockIdx.x;
    const int64_t row = part_row / p.parts;
    const int part = (int)(part_row % p.parts), keep = p.keep, begin = part * p.chunks * kChunk, end = min(begin + p.chunks * kChunk, p.vocab);
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
        return;
    }
    if (threadIdx.x == 0) s.listed = 0;

    const float* from = p.logits + row * p.row_stride;
    // Column of a thread's j-th logit of a chunk: fours of neighbours where the rows are aligned, neighbours on neighbouring lanes else.
    const auto column = [&](int chunk, int j) {
        return begin + chunk * kChunk + (aligned ? j / 4 * (kThreads * 4) + (int)threadIdx.x * 4 + j % 4 : j * kThreads + (int)threadIdx.x);
    };
    const auto load = [&](int chunk, float (&v)[values], auto read) {
        if constexpr (aligned) {
#pragma unroll
            for (int j = 0; j < values; j += 4) {
                float4 x = make_float4(kNone, kNone, kNone, kNone);
                if (column(chunk, j) < end) x = read(reinterpret_cast<const float4*>(from + column(chunk, j)));
                v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < values; ++j) v[j] = column(chunk, j) < end ? read(from + column(chunk, j)) : kNone;
        }
    };
    const auto stream = [](auto* at) { return __ldcs(at); };
    const auto again = [](auto* at) { return __ldcg(at); };

    // The running maximum and sum of this thread, and the maximum of each of its chunks; the next chunk is on its way meanwhile.
    float v[2][values], chunk_top[kMostChunks], top = kNone, sum = 0.0f;
    load(0, v[0], stream);
#pragma unroll
    for (int c = 0; c < kMostChunks; ++c) {
        chunk_top[c] = kNone;
        if (c < p.chunks) {
            if (c + 1 < kMostChunks && c + 1 < p.chunks) load(c + 1, v[(c + 1) % 2], stream);
            const float(&x)[values] = v[c % 2];
            float high[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int j = 4; j < values; j += 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) high[k] = fmaxf(high[k], x[j + k]);
            }
            chunk_top[c] = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
            const float next = fmaxf(top, chunk_top[c]), level = next > kNone ? next : 0.0f;
            float2 part_sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
            for (int j = 0; j < values; j += 2) {
                const float2 d = mul_pair(add_pair(make_float2(x[j], x[j + 1]), make_float2(-level, -level)), make_float2(kLog2e, kLog2e));
                part_sum[j / 2 % 2] = add_pair(part_sum[j / 2 % 2], make_float2(exp2_approx(d.x), exp2_approx(d.y)));
            }
            sum = sum * exp2_approx((top - level) * kLog2e) + ((part_sum[0].x + part_sum[0].y) + (part_sum[1].x + part_sum[1].y));
            top = next;
        }
    }
    // (A NaN or +inf among the logits makes the sum NaN: the maximum passes over a NaN, and inf - inf is one.)
    uint32_t warp_top_key;
    const uint32_t mine = warp_bound<kWarps>(top, keep, &warp_top_key);
    const float warp_level = from_ordered(warp_top_key);
    double total = sum * exp2_approx((top - (warp_level > kNone ? warp_level : 0.0f)) * kLog2e);
#pragma unroll
    for (int step = 16; step > 0; step /= 2) total += __shfl_xor_sync(0xffffffffu, total, step);
    if (lane == 0) {
        s.bounds[warp] = mine;
        s.tops[warp] = warp_top_key;
        s.sums[warp] = total;
    }
    __syncthreads();
    uint32_t bound_key = s.bounds[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound_key = min(bound_key, s.bounds[w]);
    const float bound = bound_key == 0 ? kNone : from_ordered(bound_key);
    uint32_t hits = 0;  // the chunks that reach the bound; they are read again, out of L2
#pragma unroll
    for (int c = 0; c < kMostChunks; ++c) hits |= (chunk_top[c] >= bound && chunk_top[c] > kNone) ? 1u << c : 0u;
    for (uint32_t rest = hits; rest != 0; rest &= rest - 1) {
        const int c = __ffs(rest) - 1;
        load(c, v[0], again);
#pragma unroll
        for (int j = 0; j < values; ++j) {
            if (v[0][j] >= bound && v[0][j] > kNone) {
                const int at = atomicAdd(&s.listed, 1);
                if (at < kPartList) s.list[at] = entry_key(v[0][j], column(c, j));
            }
        }
    }
    __syncthreads();
    const int count = s.listed;
    if (warp == kWarps - 1) {  // the part's record
        const float warp_top = lane < kWarps ? from_ordered(s.tops[lane]) : kNone;
        float part_top = warp_top;
        for (int step = 16; step > 0; step /= 2) part_top = fmaxf(part_top, __shfl_xor_sync(0xffffffffu, part_top, step));
        const float level = part_top > kNone ? part_top : 0.0f;
        double part_sum = lane < kWarps ? s.sums[lane] * exp2_approx((warp_top - level) * kLog2e) : 0.0;
        for (int step = 16; step > 0; step /= 2) part_sum += __shfl_xor_sync(0xffffffffu, part_sum, step);
        if (lane == 0) p.part_stats[part_row] = {part_sum, part_top, part_sum != part_sum};
    }
    int placed = min(count, keep);
    if (count <= kPartList) {
        for (int e = threadIdx.x; e < count; e += kThreads) {
            const uint64_t key = s.list[e];
            int place = 0;
#pragma unroll 4
            for (int k = 0; k < count; ++k) place += s.list[k] > key;
            if (place < keep) entries[place] = {from_ordered((uint32_t)(key >> 32)), (int)~(uint32_t)key};
        }
    } else {
        uint64_t last = ~0ull;
        for (placed = 0; placed < keep; ++placed) {
            uint64_t best = 0;
            for (uint32_t rest = hits; rest != 0; rest &= rest - 1) {
                const int c = __ffs(rest) - 1;
                load(c, v[0], again);
#pragma unroll
                for (int j = 0; j < values; ++j) {
                    const uint64_t key = v[0][j] > kNone ? entry_key(v[0][j], column(c, j)) : 0;
                    if (key < last) best = max(best, key);
                }
            }
            best = block_max<kWarps>(best, s.best_of);
            if (best == 0) break;
            if (threadIdx.x == 0) entries[placed] = {from_ordered((uint32_t)(best >> 32)), (int)~(uint32_t)best};
            last = best;
        }
    }
    for (int i = placed + threadIdx.x; i < keep; i += kThreads) entries[i] = {kNone, -1};
}

// A value in double precision as an integer of the same order (comparing integers is quicker), and where it is.
struct Candidate {
    uint64_t key;
    uint64_t place;  // beam << 32 | token
    __device__ __forceinline__ double value() const { return __longlong_as_double((long long)((key >> 63) ? key & 0x7fffffffffffffffull : ~key)); }
};
constexpr uint64_t kNoKey = 0x000fffffffffffffull;  // of -inf

__device__ __forceinline__ Candidate candidate_at(double value, uint64_t place) {
    const uint64_t bits = (uint64_t)__double_as_longlong(value + 0.0);  // (-0 as +0)
    return {(bits >> 63) ? ~bits : bits | 0x8000000000000000ull, place};
}

__device__ __forceinline__ bool ahead(const Candidate& a, const Candidate& b) {
    return a.key > b.key || (a.key == b.key && a.place < b.place);
}

// The value as a float, in an order that rounding keeps; what is below the lowest float counts as that, so that it stays a candidate.
__device__ __forceinline__ float as_float(double value) { return value > (double)kNone ? fmaxf((float)value, -3.402823466e38f) : kNone; }

// What other blocks have written: out of L2.
__device__ __forceinline__ BeamEntry load_entry(const BeamEntry* at) {
    const float2 two = __ldcg(reinterpret_cast<const float2*>(at));
    return {two.x, __float_as_int(two.y)};
}
__device__ __forceinline__ BeamPart load_part(const BeamPart* at) {
    const double2 two = __ldcg(reinterpret_cast<const double2*>(at));
    return {two.x, __int_as_float(__double2loint(two.y)), __double2hiint(two.y)};
}

struct GroupShared {
    double base[kMostSelectBeams];  // score - normaliser; -inf: the beam offers nothing
    Candidate list[kGroupList], best_of[kWarps];
    uint32_t bounds[kWarps];
    int listed, not_finite;
};

__device__ __forceinline__ void best_of_group(const BeamSelectParams& p, GroupShared& s, int64_t group) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, keep = p.keep;
    if (threadIdx.x == 0) s.listed = 0, s.not_finite = 0;
    // The lists' first entries, the best of all lists, then the second ones and so on, are asked for ahead of the normalisers and
    // kept.  Every eight neighbours go to the eight warps in an order that changes: the bound is good where each warp has its
    // share of the best, and one beam's lists are neighbours.
    const BeamEntry* entries = p.entries + group * p.beams * p.parts * keep;
    const int lists = p.beams * p.parts;
    constexpr int kHeld = kHeldEntries * kThreads;
    const int all_held = min(lists * keep, kHeld);
    BeamEntry held[kHeldEntries];
    int held_list[kHeldEntries];
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        const uint32_t y = i * 32 + lane;
        const int x = (int)(y * 8 + ((warp + (y * 2654435761u >> 29)) & 7)), slot = (int)p.by_lists.quotient(x);
        held_list[i] = x - slot * lists;
        held[i] = x < all_held ? load_entry(entries + held_list[i] * keep + slot) : BeamEntry{kNone, -1};
    }
    __syncthreads();
    for (int b = warp; b < p.beams; b += kWarps) {
        const int64_t row = group * p.beams + b;
        const BeamPart* parts = p.part_stats + row * p.parts;
        const float score = p.scores[row];
        const bool ended = p.finished && p.finished[row];
        float top = kNone;
        double sum = 0.0;
        int wrong = !(score < -kNone);
        for (int first = 0; first < p.parts; first += 64) {  // (two a lane: one trip to memory where the parts are few)
            BeamPart part[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = first + i * 32 + lane;
                part[i] = at < p.parts ? load_part(parts + at) : BeamPart{0.0, kNone, 0};
                wrong |= part[i].not_finite;
            }
            float next = fmaxf(top, fmaxf(part[0].top, part[1].top));
            for (int step = 16; step > 0; step /= 2) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, step));
            const float level = next > kNone ? next : 0.0f;
            sum *= exp2_approx((top - level) * kLog2e);
#pragma unroll
            for (int i = 0; i < 2; ++i) sum += part[i].sum * exp2_approx((part[i].top - level) * kLog2e);
            top = next;
        }
        for (int step = 16; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
        wrong = __any_sync(0xffffffffu, wrong);
        if (lane == 0) {
            if (wrong) s.not_finite = 1;
            s.base[b] = ended ? (double)score : sum > 0.0 ? (double)score - ((double)top + log_of(sum)) : (double)kNone;
        }
    }
    __syncthreads();
    const auto candidate_of = [&](int of_list, BeamEntry entry) {
        const int b = (int)p.by_parts.quotient(of_list);
        return candidate_at(s.base[b] + (double)entry.logit, (uint64_t)b << 32 | (uint32_t)entry.token);
    };
    float largest = kNone;
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        largest = fmaxf(largest, as_float(candidate_of(held_list[i], held[i]).value()));
    }
    const uint32_t mine = warp_bound<kWarps>(largest, keep, nullptr);
    if (lane == 0) s.bounds[warp] = mine;
    __syncthreads();
    uint32_t bound_key = s.bounds[0];
    for (int w = 1; w < kWarps; ++w) bound_key = min(bound_key, s.bounds[w]);
    const float bound = bound_key == 0 ? kNone : from_ordered(bound_key);
    // (rounding to float keeps the order: what is at or above the bound in double is so in float)
    const auto offer = [&](const Candidate& c) {
        if (!(c.key > kNoKey && as_float(c.value()) >= bound)) return false;
        const int at = atomicAdd(&s.listed, 1);
        if (at < kGroupList) s.list[at] = c;
        return true;
    };
    if (largest >= bound && largest > kNone) {
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) {
            offer(candidate_of(held_list[i], held[i]));
        }
    }
    if (all_held < lists * keep) {  // lists are in order: each from where it is not held on, as far as it reaches the bound
        for (int q = threadIdx.x; q < lists; q += kThreads) {
            for (int slot = max(kHeld - q + lists - 1, 0) / lists; slot < keep && offer(candidate_of(q, load_entry(entries + q * keep + slot))); ++slot) {
            }
        }
    }
    __syncthreads();
    const int count = s.listed;
    const bool wrong = s.not_finite != 0;
    int placed = wrong ? 0 : min(count, keep);
    const auto put = [&](int place, const Candidate& c) {
        const int64_t at = group * keep + place;
        p.out_scores[at] = as_float(c.value());
        p.parents[at] = (int64_t)(c.place >> 32);
        p.tokens[at] = (int64_t)(uint32_t)c.place;
    };
    if (wrong) {
    } else if (count <= kGroupList) {
        for (int e = threadIdx.x; e < count; e += kThreads) {
            const Candidate c = s.list[e];
            int place = 0;
#pragma unroll 4
            for (int k = 0; k < count; ++k) place += ahead(s.list[k], c);
            if (place < keep) put(place, c);
        }
    } else {  // more that tie at the bound than the list holds: sweep after sweep, the best that is behind the last one
        Candidate last{~0ull, 0};
        for (placed = 0; placed < keep; ++placed) {
            Candidate best{kNoKey, ~0ull};
            for (int e = threadIdx.x; e < lists * keep; e += kThreads) {
                const Candidate c = candidate_of(e / keep, load_entry(entries + e));
                if (ahead(last, c) && ahead(c, best)) best = c;
            }
            for (int step = 16; step > 0; step /= 2) {
                const Candidate other{__shfl_xor_sync(0xffffffffu, best.key, step), __shfl_xor_sync(0xffffffffu, best.place, step)};
                if (ahead(other, best)) best = other;
            }
            if (lane == 0) s.best_of[warp] = best;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w) {
                if (ahead(s.best_of[w], best)) best = s.best_of[w];
            }
            __syncthreads();
            if (best.key == kNoKey) break;
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

template <int values, bool aligned>
__global__ void __launch_bounds__(kThreads, values == 16 ? 4 : 2) beam_select_kernel(const __grid_constant__ BeamSelectParams p) {
    __shared__ union Shared {
        PartShared part;
        GroupShared group;
        __device__ Shared() {}
    } shared;
    __shared__ int is_last;
    part_of_row<values, aligned>(p, shared.part);
    const int64_t group = blockIdx.x / (unsigned)(p.beams * p.parts);
    __syncthreads();
    if (threadIdx.x == 0) {  // (release: the block's part, ordered before by the barrier; acquire: the others')
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + group) : "memory");
        is_last = before == p.beams * p.parts - 1;
        if (is_last) p.arrived[group] = 0;
    }
    __syncthreads();
    if (is_last) best_of_group(p, shared.group, group);
}

}  // namespace

Quotients::Quotients(uint32_t by) : one(by == 1), magic((uint32_t)(((uint64_t(1) << 32) + by - 1) / by)) {}

void plan_beam_select(BeamSelectParams& p, int sm_count) {
    const int64_t rows = p.groups * p.beams;
    // Long parts cost least per logit (what a part costs besides is shared by up to eight chunks of 4096); where they would be
    // fewer than the GPU holds at once, shorter ones spread the rows further.
    const auto chunks = [&](int values) { return (p.vocab + kThreads * values - 1) / (kThreads * values); };
    p.values = rows * chunks(16) < sm_count ? 4 : 16;
    const int all = chunks(p.values);
    p.chunks = kMostChunks;
    while (p.chunks > 1 && rows * ((all + p.chunks - 1) / p.chunks) < 2 * sm_count) --p.chunks;
    p.parts = (all + p.chunks - 1) / p.chunks;
    p.chunks = (all + p.parts - 1) / p.parts;  // (no part much shorter than the others)
    p.by_parts = Quotients((uint32_t)p.parts);
    p.by_lists = Quotients((uint32_t)(p.beams * p.parts));
    p.aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.row_stride % 4 == 0 && p.vocab % 4 == 0;
}

cudaError_t launch_beam_select(const BeamSelectParams& p, cudaStream_t stream) {
    const unsigned blocks = (unsigned)(p.groups * p.beams * p.parts);
    if (p.values == 4) {
        if (p.aligned) beam_select_kernel<4, true><<<blocks, kThreads, 0, stream>>>(p);
        else beam_select_kernel<4, false><<<blocks, kThreads, 0, stream>>>(p);
    } else {
        if (p.aligned) beam_select_kernel<16, true><<<blocks, kThreads, 0, stream>>>(p);
        else beam_select_kernel<16, false><<<blocks, kThreads, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace psx
