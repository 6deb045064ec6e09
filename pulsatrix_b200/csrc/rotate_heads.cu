// Queries and keys on their way from a projection into the attention, in one pass: a norm per head, the rotation by the position, and keys
// and values into the pages of the cache.
//
//     y = x / sqrt(mean(x^2) + eps) * w,   (u, v) -> (u cos a - v sin a, v cos a + u sin a) for pair j with a = position * frequency_j
//
// in floats, rounded once at the end.  The angle is taken in double precision, in quarter turns: position * frequency * 2 / pi less the
// nearest whole number is what is left for sincospif, an eighth of a turn at most, so that its rounding to a float counts 2^-26 quarter turns
// however far the position is (in floats, an angle of 100,000 is off by up to 4e-3).
//
// A lane holds eight dimensions of a head, as two runs of four: of both halves where pairs are (j, j + rotated / 2), neighbours where they
// are (2 j, 2 j + 1) and where dimensions are not rotated; so both elements of a pair are in one lane, which makes eight to 32 lanes a head.
// A warp has a position, or some heads of one where positions are few: the row that it belongs to, its page and its angles are found once for
// all of its heads.  Bound by HBM for prompts, by latency for single positions.
#include "rotate_heads.cuh"

#include <algorithm>
#include <type_traits>

#include "elements.cuh"

namespace psx {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kAhead = 4;  // heads of a lane that are on their way at once
constexpr int kRowOk = 0, kRowCacheFull = 64, kRowBadOffsets = 65;  // (psx_row_status)

// Four elements as they come.
template <class T>
struct Run {
    using Bits = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
    Bits bits;
    __device__ __forceinline__ void to_floats(float (&x)[4]) const {
        T e[4];
        __builtin_memcpy(e, &bits, sizeof(e));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = to_float(e[i]);
    }
    __device__ __forceinline__ static Run of(const float (&x)[4]) {
        const T e[4] = {from_float<T>(x[0]), from_float<T>(x[1]), from_float<T>(x[2]), from_float<T>(x[3])};
        Run r;
        __builtin_memcpy(&r.bits, e, sizeof(e));
        return r;
    }
    __device__ __forceinline__ static Run at(const T* p) { return {__ldcs(reinterpret_cast<const Bits*>(p))}; }
    __device__ __forceinline__ void put(T* p) const { *reinterpret_cast<Bits*>(p) = bits; }
};

// What a row of the batch may store.
__device__ __forceinline__ int row_status(const RotateHeadsParams& p, int row) {
    const int64_t begin = p.offsets[row], end = p.offsets[row + 1], first = p.first[row];
    if (begin < 0 || end < begin || end > p.total || first < 0) return kRowBadOffsets;
    if (!p.cache.keys) return kRowOk;
    const int64_t length = p.cache.table.length(row);
    return first > length || end - begin > length - first ? kRowCacheFull : kRowOk;
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

template <class T, int lanes>
__global__ void __launch_bounds__(kThreads) rotate_heads_kernel(const __grid_constant__ RotateHeadsParams p) {
    constexpr int kSlots = 32 / lanes;  // heads of a warp at once
    const int lane = threadIdx.x % 32, l = lane % lanes, slot = lane / lanes;
    if (p.row_status) {
        for (int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x; row < p.batch; row += (int64_t)gridDim.x * kThreads) p.row_status[row] = row_status(p, (int)row);
    }
    const int64_t unit = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    if (unit >= p.total * p.slabs) return;
    const int64_t token = unit / p.slabs;
    const int dims = p.head_dim, all = p.heads + p.kv_heads + (p.cache.keys ? p.kv_heads : 0);
    const int begin = (int)(unit % p.slabs) * p.slab_rows, end = min(begin + p.slab_rows, all);
    const bool here = 8 * l < dims, turns = 8 * l < p.rotated, halves = turns && !p.interleaved;
    const int low = halves ? 4 * l : 8 * l, high = halves ? 4 * l + p.rotated / 2 : 8 * l + 4;

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

    float cosine[4], sine[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        cosine[j] = 1.0f, sine[j] = 0.0f;
        if (turns) {
            const double quarters = (double)position * (p.frequencies[4 * l + j] * 0.63661977236758134308);
            const double whole = rint(quarters);
            sincospif((float)(quarters - whole) * 0.5f, &sine[j], &cosine[j]);
            const int quadrant = (int)((long long)whole & 3);
            if (quadrant & 1) {
                const float c = cosine[j];
                cosine[j] = -sine[j];
                sine[j] = c;
            }
            if (quadrant & 2) cosine[j] = -cosine[j], sine[j] = -sine[j];
        }
    }
    for (int r0 = begin; r0 < end; r0 += kAhead * kSlots) {
        Run<T> a[kAhead], b[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int r = r0 + i * kSlots + slot;
            a[i].bits = b[i].bits = {};
            if (r < end && here) {
                const T* from = r < p.heads ? static_cast<const T*>(p.q) + token * p.q_stride + (int64_t)r * dims
                    : r < p.heads + p.kv_heads ? static_cast<const T*>(p.k) + token * p.k_stride + (int64_t)(r - p.heads) * dims
                                               : static_cast<const T*>(p.v) + token * p.v_stride + (int64_t)(r - p.heads - p.kv_heads) * dims;
                a[i] = Run<T>::at(from + low);
                b[i] = Run<T>::at(from + high);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int r = r0 + i * kSlots + slot;
            const bool is_query = r < p.heads, is_value = r >= p.heads + p.kv_heads;
            const T* weight = static_cast<const T*>(is_query ? p.q_weight : p.k_weight);
            float x[4], y[4];
            a[i].to_floats(x);
            b[i].to_floats(y);
            if (p.q_weight || p.k_weight) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) sum += x[j] * x[j] + y[j] * y[j];
#pragma unroll
                for (int step = 1; step < lanes; step *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
                if (weight && here) {
                    const float scale = 1.0f / sqrtf(sum / (float)dims + p.eps);
                    const float4 wx = load_four(weight + low), wy = load_four(weight + high);
                    x[0] *= scale * wx.x, x[1] *= scale * wx.y, x[2] *= scale * wx.z, x[3] *= scale * wx.w;
                    y[0] *= scale * wy.x, y[1] *= scale * wy.y, y[2] *= scale * wy.z, y[3] *= scale * wy.w;
                }
            }
            if (r >= end || !here) continue;
            if (is_value) {  // (bit by bit)
                if (place >= 0) {
                    T* to = reinterpret_cast<T*>(p.cache.values) + place + (r - p.heads - p.kv_heads) * head_step;
                    a[i].put(to + low);
                    b[i].put(to + high);
                }
                continue;
            }
            float u[4], w[4];
            if (!p.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[j] = x[j] * cosine[j] - y[j] * sine[j];
                    w[j] = y[j] * cosine[j] + x[j] * sine[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    u[2 * j] = x[2 * j] * cosine[j] - x[2 * j + 1] * sine[j];
                    u[2 * j + 1] = x[2 * j + 1] * cosine[j] + x[2 * j] * sine[j];
                    w[2 * j] = y[2 * j] * cosine[2 + j] - y[2 * j + 1] * sine[2 + j];
                    w[2 * j + 1] = y[2 * j + 1] * cosine[2 + j] + y[2 * j] * sine[2 + j];
                }
            }
            if (!turns) {  // (a product with 0 would make an infinity's neighbour NaN)
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = x[j], w[j] = y[j];
            }
            const Run<T> first = Run<T>::of(u), second = Run<T>::of(w);
            if (is_query) {
                T* to = static_cast<T*>(p.q_out) + (token * p.heads + r) * dims;
                first.put(to + low);
                second.put(to + high);
            } else {
                if (p.k_out) {
                    T* to = static_cast<T*>(p.k_out) + (token * p.kv_heads + (r - p.heads)) * dims;
                    first.put(to + low);
                    second.put(to + high);
                }
                if (place >= 0) {
                    T* to = reinterpret_cast<T*>(p.cache.keys) + place + (r - p.heads) * head_step;
                    first.put(to + low);
                    second.put(to + high);
                }
            }
        }
    }
}

template <class T>
cudaError_t launch(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    const int lanes = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32, slots = 32 / lanes;
    const int all = p.heads + p.kv_heads + (p.cache.keys ? p.kv_heads : 0);
    // A warp per position where that fills the GPU, or as many as there are heads to share out.
    const int64_t wanted = std::max<int64_t>(1, (int64_t)sm_count * 32 / std::max<int64_t>(p.total, 1));
    const int64_t most = (all + slots - 1) / slots;
    p.slabs = (int)std::min(wanted, most);
    p.slab_rows = ((all + p.slabs - 1) / p.slabs + slots - 1) / slots * slots;
    const int64_t blocks = std::max<int64_t>(1, (p.total * p.slabs + kWarps - 1) / kWarps);
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    if (lanes == 8) rotate_heads_kernel<T, 8><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
    else if (lanes == 16) rotate_heads_kernel<T, 16><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
    else rotate_heads_kernel<T, 32><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rotate_heads(RotateHeadsParams& p, int sm_count, cudaStream_t stream) {
    if (p.type == kFloat32) return launch<float>(p, sm_count, stream);
    if (p.type == kBfloat16) return launch<__nv_bfloat16>(p, sm_count, stream);
    return launch<__half>(p, sm_count, stream);
}

}  // namespace psx
