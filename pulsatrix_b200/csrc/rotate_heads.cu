// Queries and keys on their way from a projection into the attention, in one pass: a norm per head, the rotation by the position, and keys
// and values into the pages of the cache.
//
//     y = x / sqrt(mean(x^2) + eps) * w,   (u, v) -> (u cos a - v sin a, v cos a + u sin a) for pair j with a = position * frequency_j
//
// in floats, rounded once at the end.  The angle is taken in double precision, in quarter turns: position * frequency * 2 / pi less the
// nearest whole number is what is left, an eighth of a turn at most, pi / 4 radians, so that its rounding to a float counts 2^-25 radians at most,
// however far the position is (in floats, an angle of 100,000 is off by up to 4e-3).
//
// A lane holds two runs of 16 bytes of a head (of 8, where half of the rotated dimensions is not a multiple of 16 bytes): one of both halves where pairs are
// (j, j + rotated / 2), neighbours where they are (2 j, 2 j + 1) and where dimensions are not rotated; so both elements of a pair are in one
// lane, and four to 32 lanes have a head.  A warp has a position, or some heads of one where positions are few: the row that it belongs to, its page and
// its angles, which the lanes share out and pass on through shared memory, are found once for all of its heads.  Bound by HBM for prompts, by latency for
// single positions: 12 prompts of up to 2111 positions, 32 + 8 + 8 heads of 128, take 94 us in bf16 (5.7 TB/s), 171 in fp32 (6.3 TB/s).
#include "rotate_heads.cuh"

#include <algorithm>
#include <type_traits>

#include "elements.cuh"
#include "psx_device.cuh"

namespace psx {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kAhead = 2;  // heads of a lane that are on their way at once
constexpr int kMostPairs = 128;
constexpr int kRowOk = 0, kRowCacheFull = 64, kRowBadOffsets = 65;  // (psx_row_status)

// `count` elements as they come.
template <class T, int count>
struct Run {
    using Bits = typename std::conditional<sizeof(T) * count == 16, uint4, uint2>::type;
    Bits bits;
    __device__ __forceinline__ void to_floats(float (&x)[count]) const {
        T e[count];
        __builtin_memcpy(e, &bits, sizeof(e));
#pragma unroll
        for (int i = 0; i < count; ++i) x[i] = to_float(e[i]);
    }
    __device__ __forceinline__ static Run of(const float (&x)[count]) {
        T e[count];
#pragma unroll
        for (int i = 0; i < count; ++i) e[i] = from_float<T>(x[i]);
        Run r;
        __builtin_memcpy(&r.bits, e, sizeof(e));
        return r;
    }
    __device__ __forceinline__ static Run at(const T* p) { return {*reinterpret_cast<const Bits*>(p)}; }
    __device__ __forceinline__ void put(T* p) const { *reinterpret_cast<Bits*>(p) = bits; }
};

// 1 / sqrt(x), the function's two units brought to one by a step of Newton's method.
__device__ __forceinline__ float inverse_root(float x) {
    const float y = rsqrtf(x);
    const float better = fmaf(y, fmaf(-0.5f * x * y, y, 0.5f), y);
    return x > 0.0f && x < __builtin_huge_valf() ? better : y;  // (0 and infinity: inf * 0 in the step)
}

// What a row of the batch may store.
__device__ __forceinline__ int row_status(const RotateHeadsParams& p, int row) {
    const int64_t begin = p.offsets[row], end = p.offsets[row + 1], first = p.first[row];
    if (begin < 0 || end < begin || end > p.total || first < 0) return kRowBadOffsets;
    if (!p.cache.keys) return kRowOk;
    const int64_t length = p.cache.table.length(row);
    return first > length || end - begin > length - first ? kRowCacheFull : kRowOk;
}

// Sine and cosine of an eighth of a turn at most, by their power series: what is left out is below 2.2e-9 and 1.2e-10.
__device__ __forceinline__ void sine_and_cosine(float x, float& sine, float& cosine) {
    const float z = x * x;
    sine = fmaf(x, z * fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
}

// Heads of one operand on their way into L2, their lines shared out over the warp's lanes.
template <class T>
__device__ __forceinline__ void ask_for(const T* from, int heads, int dims) {
    const char* at = reinterpret_cast<const char*>(from);
    for (int line = (threadIdx.x % 32) * 128; line < heads * dims * (int)sizeof(T); line += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + line));
}

// The row that position `at` of the packed ones belongs to; -1: none.  The warp looks at 32 offsets at a time.
__device__ __forceinline__ int row_of(const int64_t* offsets, int batch, int64_t at) {
    const int lane = threadIdx.x % 32;
    int low = 0, count = batch + 1;  // offsets[low .. low + count) hold the last one that is not above
    while (true) {
        const int step = (count + 31) / 32, probe = lane * step;
        const unsigned reached = __ballot_sync(0xffffffffu, probe < count && offsets[low + min(probe, count - 1)] <= at);
        const int found = __popc(reached) - 1;
        if (found < 0) return -1;
        low += found * step;
        count = min(step, count - found * step);
        if (count <= 1) break;
    }
    return low < batch && offsets[low] <= at && at < offsets[low + 1] ? low : -1;
}

template <class T, int run, int lanes>
__global__ void __launch_bounds__(kThreads, run == 8 ? 5 : 6) rotate_heads_kernel(const __grid_constant__ RotateHeadsParams p) {
    using R = Run<T, run>;
    constexpr int kSlots = 32 / lanes;  // heads of a warp at once
    constexpr int kPairs = run;         // of a lane
    __shared__ __align__(16) float2 turned[kWarps][kMostPairs];  // cosine and sine of every pair
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % lanes, slot = lane / lanes;
    grid_dependency_wait();
    grid_dependents_may_launch();
    if (p.row_status) {
        for (int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x; row < p.batch; row += (int64_t)gridDim.x * kThreads) p.row_status[row] = row_status(p, (int)row);
    }
    const unsigned unit = blockIdx.x * kWarps + warp, position_of = p.slabs == 1 ? unit : unit / (unsigned)p.slabs;
    if (position_of >= (unsigned)p.total) return;
    const int64_t token = position_of;
    const int dims = p.head_dim, all = p.heads + p.kv_heads + (p.cache.keys ? p.kv_heads : 0);
    const int begin = (int)(unit - position_of * (unsigned)p.slabs) * p.slab_rows, end = min(begin + p.slab_rows, all);
    const bool turns = 2 * run * l < p.rotated, halves = turns && !p.interleaved;
    const int low = halves ? run * l : 2 * run * l, high = halves ? run * l + p.rotated / 2 : 2 * run * l + run;
    const bool low_here = low < dims && 2 * run * l < dims, high_here = high < dims && 2 * run * l < dims;

    // What does not depend on the row is asked for before it is known: the position's heads on their way into L2, the frequencies into registers.
    const T* const q_at = static_cast<const T*>(p.q) + token * p.q_stride;
    const T* const k_at = static_cast<const T*>(p.k) + token * p.k_stride;
    const T* const v_at = static_cast<const T*>(p.v) + (p.cache.keys ? token * p.v_stride : 0);
    const int first_key = max(begin - p.heads, 0), last_key = min(end - p.heads, p.kv_heads);
    const int first_value = max(begin - p.heads - p.kv_heads, 0), last_value = end - p.heads - p.kv_heads;
    // (Not for fp32, which has twice the bytes of a lane on their way as it is, 172 us would become 205 below; nor for few heads, 16 + 4 + 4 of 64 dimensions 21 us and
    // 23; but 32 + 8 + 8 of them 58 without and 52.)
    if (sizeof(T) == 2 && (end - begin) * dims >= 2048) {
        ask_for(q_at + begin * dims, min(end, p.heads) - begin, dims);
        ask_for(k_at + first_key * dims, last_key - first_key, dims);
        ask_for(v_at + first_value * dims, last_value - first_value, dims);
    }
    double frequency[kMostPairs / 32];
#pragma unroll
    for (int i = 0; i < kMostPairs / 32; ++i) frequency[i] = i * 32 + lane < p.rotated / 2 ? p.frequencies[i * 32 + lane] : 0.0;

    const int row = row_of(p.offsets, p.batch, token);
    if (row < 0) return;
    const int64_t position = (int64_t)((uint64_t)p.first[row] + (uint64_t)(token - p.offsets[row]));
    int64_t place = -1;  // of head 0 in the pages
    if (p.cache.keys && row_status(p, row) == kRowOk) {
        const PageTableView& t = p.cache.table;
        const int page = t.pages[(int64_t)row * t.max_pages + (position >> t.shift)];
        if (t.real(page)) place = ((int64_t)page * p.kv_heads * t.page_size + (position & (t.page_size - 1))) * dims;
    }
    const int64_t head_step = (int64_t)p.cache.table.page_size * dims;

#pragma unroll
    for (int i = 0; i < kMostPairs / 32; ++i) {
        const int j = i * 32 + lane;
        if (j >= p.rotated / 2) continue;
        // Quarter turns and the nearest whole number of them: added to 1.5 * 2^52 it is rounded to a whole number, and its last bits are the sum's (for less
        // than 2^51 of them).
        const double quarters = (double)position * (frequency[i] * 0.63661977236758134308), shifted = quarters + 6755399441055744.0;
        const int quadrant = __double2loint(shifted);
        float sine, cosine;
        sine_and_cosine((float)((quarters - (shifted - 6755399441055744.0)) * 1.57079632679489661923), sine, cosine);
        float2 turn = quadrant & 1 ? make_float2(-sine, cosine) : make_float2(cosine, sine);
        if (quadrant & 2) turn = make_float2(-turn.x, -turn.y);
        turned[warp][j] = turn;
    }
    __syncwarp();
    float cosine[kPairs], sine[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; j += 2) {
        float4 two = make_float4(1.0f, 0.0f, 1.0f, 0.0f);
        if (turns) two = *reinterpret_cast<const float4*>(&turned[warp][run * l + j]);
        cosine[j] = two.x, sine[j] = two.y, cosine[j + 1] = two.z, sine[j + 1] = two.w;
    }

    // Heads first .. last of one operand, `from` being its head 0 at this position.
    const auto heads_of = [&](const T* from, int first, int last, const T* weight, auto put) {
        float wx[run], wy[run];
#pragma unroll
        for (int j = 0; j < run; ++j) wx[j] = wy[j] = 1.0f;
        if (weight) {
            if (low_here) R::at(weight + low).to_floats(wx);
            if (high_here) R::at(weight + high).to_floats(wy);
        }
#pragma unroll 1
        for (int h0 = first; h0 < last; h0 += kAhead * kSlots) {
            R a[kAhead], b[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int h = h0 + i * kSlots + slot;
                a[i].bits = b[i].bits = {};
                if (h < last && low_here) a[i] = R::at(from + h * dims + low);
                if (h < last && high_here) b[i] = R::at(from + h * dims + high);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (h0 + i * kSlots >= last) continue;  // (the warp together)
                const int h = h0 + i * kSlots + slot;
                float x[run], y[run];
                a[i].to_floats(x);
                b[i].to_floats(y);
                if (weight) {
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < run; ++j) sum += x[j] * x[j] + y[j] * y[j];
#pragma unroll
                    for (int step = 1; step < lanes; step *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
                    const float scale = inverse_root(sum * p.inverse_dims + p.eps);
#pragma unroll
                    for (int j = 0; j < run; ++j) x[j] *= scale * wx[j], y[j] *= scale * wy[j];
                }
                if (turns) {  // (elsewhere a product with 0 would make an infinity's neighbour NaN)
                    if (!p.interleaved) {
#pragma unroll
                        for (int j = 0; j < run; ++j) {
                            const float u = x[j] * cosine[j] - y[j] * sine[j];
                            y[j] = y[j] * cosine[j] + x[j] * sine[j];
                            x[j] = u;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < run / 2; ++j) {
                            const float u = x[2 * j] * cosine[j] - x[2 * j + 1] * sine[j], w = y[2 * j] * cosine[run / 2 + j] - y[2 * j + 1] * sine[run / 2 + j];
                            x[2 * j + 1] = x[2 * j + 1] * cosine[j] + x[2 * j] * sine[j];
                            y[2 * j + 1] = y[2 * j + 1] * cosine[run / 2 + j] + y[2 * j] * sine[run / 2 + j];
                            x[2 * j] = u, y[2 * j] = w;
                        }
                    }
                }
                if (h < last) put(h, R::of(x), R::of(y));
            }
        }
    };
    const auto put_at = [&](T* to, const R& a, const R& b) {
        if (low_here) a.put(to + low);
        if (high_here) b.put(to + high);
    };
    if (begin < p.heads) {
        T* to = static_cast<T*>(p.q_out) + token * p.heads * dims;
        heads_of(q_at, begin, min(end, p.heads), static_cast<const T*>(p.q_weight),
                 [&](int h, const R& a, const R& b) { put_at(to + h * dims, a, b); });
    }
    if (first_key < last_key) {
        T* to = static_cast<T*>(p.k_out) + token * p.kv_heads * dims;
        T* pages = reinterpret_cast<T*>(p.cache.keys) + place;
        heads_of(k_at, first_key, last_key, static_cast<const T*>(p.k_weight), [&](int h, const R& a, const R& b) {
            if (p.k_out) put_at(to + h * dims, a, b);
            if (place >= 0) put_at(pages + h * head_step, a, b);
        });
    }
    if (place >= 0 && first_value < last_value) {  // (bit by bit)
        const T* from = v_at;
        T* pages = reinterpret_cast<T*>(p.cache.values) + place;
#pragma unroll 1
        for (int h0 = first_value; h0 < last_value; h0 += kAhead * kSlots) {
            R a[kAhead], b[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int h = h0 + i * kSlots + slot;
                if (h < last_value && low_here) a[i] = R::at(from + h * dims + low);
                if (h < last_value && high_here) b[i] = R::at(from + h * dims + high);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int h = h0 + i * kSlots + slot;
                if (h < last_value) put_at(pages + h * head_step, a[i], b[i]);
            }
        }
    }
}

template <class T, int run, int lanes>
cudaError_t launch_lanes(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    constexpr int slots = 32 / lanes;
    const int all = p.heads + p.kv_heads + (p.cache.keys ? p.kv_heads : 0);
    // A warp per position where that fills the GPU, or as many as there are heads to share out.  (Two a position: 108 us instead of 101 in the case
    // below; a warp for two to five positions one after the other: 144 to 182.)
    const int64_t wanted = std::max<int64_t>(1, (int64_t)sm_count * 32 / std::max<int64_t>(p.total, 1));
    const int64_t most = (all + slots - 1) / slots;
    p.slabs = (int)std::min(wanted, most);
    p.slab_rows = ((all + p.slabs - 1) / p.slabs + slots - 1) / slots * slots;
    const int64_t blocks = std::max<int64_t>(1, (p.total * p.slabs + kWarps - 1) / kWarps);
    if (blocks * kWarps > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_overlapping(rotate_heads_kernel<T, run, lanes>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
}

template <class T, int run>
cudaError_t launch_run(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    const int lanes = (p.head_dim + 2 * run - 1) / (2 * run);
    if constexpr (run == 8) {
        if (lanes <= 4) return launch_lanes<T, run, 4>(p, sm_count, stream);
    }
    if (lanes <= 8) return launch_lanes<T, run, 8>(p, sm_count, stream);
    if (run == 8 || lanes <= 16) return launch_lanes<T, run, 16>(p, sm_count, stream);
    return launch_lanes<T, run, 32>(p, sm_count, stream);
}

template <class T>
cudaError_t launch(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    p.inverse_dims = 1.0f / (float)p.head_dim;
    if constexpr (sizeof(T) == 2) {
        // (12 prompts of up to 2111, 40 heads of 128 and 8 more for the values: 98 us with runs of 16 bytes, 213 with 8)
        if (p.rotated % 16 == 0) return launch_run<T, 8>(p, sm_count, stream);
    }
    return launch_run<T, 4>(p, sm_count, stream);
}

}  // namespace

cudaError_t launch_rotate_heads(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    if (p.type == kFloat32) return launch<float>(p, sm_count, stream);
    if (p.type == kBfloat16) return launch<__nv_bfloat16>(p, sm_count, stream);
    return launch<__half>(p, sm_count, stream);
}

}  // namespace psx
