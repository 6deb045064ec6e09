// New keys and values on their way into a cache held in 8 bits.
//
// A block of `block` positions of a (row, kv head) has one scale, a power of two: the least 2^e at which the block's largest
// magnitude, 448 * 2^e at most, has a code.  Codes are floating point themselves (e4m3), so a finer scale would buy no
// precision, and with powers of two nothing is rounded but the codes: values / scale is exact, and when a block that is
// partly filled has to grow its scale, the old codes times 2^(old - new) are exact too unless they fall below the smallest
// normal code.  A decoding step that adds one position at a time ends with what one call with all of them leaves, but for
// those.
//
// A block of 1 to 8 warps takes (block of positions, kv head, keys or values): it holds the elements in registers, 64 a thread,
// between the maximum and the codes, so that the input is read once and some 160 KB per SM are on their way.  Bound by HBM for
// prompts, by latency for single positions.
#include "store_cache_8bit.cuh"

#include <algorithm>

#include "elements.cuh"
#include "row_prefix.cuh"

namespace psx {
namespace {

constexpr int kHeld = 64;  // elements of a block that a thread holds

struct NewRows {
    int64_t begin, count, cached;
    int32_t status;
};

// A row whose offsets or positions do not fit has nothing stored.
__device__ __forceinline__ NewRows new_rows(const StoreCacheParams& p, int64_t row) {
    const int64_t begin = p.offsets[row], end = p.offsets[row + 1], cached = p.cached[row];
    if (begin < 0 || end < begin || end > p.total || cached < 0) return {0, 0, 0, kRowBadOffsets};
    if (cached > p.cache.max_len || end - begin > p.cache.max_len - cached) return {0, 0, 0, kRowCacheFull};
    return {begin, end - begin, cached, kRowOk};
}

// The power of two that is the scale of a block whose largest magnitude is `largest`, finite.  448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_of(float largest) {
    const uint32_t bits = __float_as_uint(largest);
    const int exponent = (int)(bits >> 23) - 127;  // (0 and subnormal magnitudes: -127)
    const int e = exponent - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// Sixteen bytes of the new elements, as they come.
template <class T>
struct Vector {
    static constexpr int elements = 16 / sizeof(T);
    uint4 bits;

    __device__ __forceinline__ float operator[](int i) const {
        const uint32_t words[4] = {bits.x, bits.y, bits.z, bits.w};
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(words[i]);
        } else {
            const unsigned short half = (unsigned short)(words[i / 2] >> (i % 2 * 16));
            T x;
            __builtin_memcpy(&x, &half, 2);
            return to_float(x);
        }
    }
    // Elements i .. i + 3 times `inverse` as codes.
    __device__ __forceinline__ uint32_t codes(int i, float inverse) const {
        return floats_to_codes((*this)[i] * inverse, (*this)[i + 1] * inverse) | floats_to_codes((*this)[i + 2] * inverse, (*this)[i + 3] * inverse) << 16;
    }
    // The larger magnitudes, as bit patterns (of their size, numbers without a sign are in order; two side by side for 16 bits).
    static __device__ __forceinline__ uint32_t larger(uint32_t most, const uint4& x) {
        for (const uint32_t w : {x.x, x.y, x.z, x.w}) {
            if constexpr (sizeof(T) == 4) most = max(most, w & 0x7fffffffu);
            else most = __vmaxu2(most, w & 0x7fff7fffu);
        }
        return most;
    }
    // The larger of the patterns as a float's.
    static __device__ __forceinline__ uint32_t magnitude(uint32_t most) {
        if constexpr (sizeof(T) == 4) {
            return most;
        } else {
            const unsigned short half = (unsigned short)max(most & 0xffffu, most >> 16);
            T x;
            __builtin_memcpy(&x, &half, 2);
            return __float_as_uint(to_float(x)) & 0x7fffffffu;
        }
    }
};

// Threads: the elements of a block of positions over kHeld.
template <class T, int threads>
__global__ void __launch_bounds__(threads, 512 / threads) store_cache_8bit_kernel(const __grid_constant__ StoreCacheParams p) {
    using V = Vector<T>;
    constexpr int kWarps = threads / 32, kVectors = kHeld / V::elements;
    extern __shared__ int prefix[];
    __shared__ int carry[kWarps];
    __shared__ uint32_t largest_of[2][kWarps];
    const Cache8bitView& c = p.cache;
    const int batch = (int)c.batch, block = c.block, per_row = c.head_dim / V::elements;
    sum_of_rows(batch, prefix, carry, [&](int row) {
        const NewRows r = new_rows(p, row);
        if (p.row_status && blockIdx.x == 0) p.row_status[row] = r.status;
        return r.count ? (int)((r.cached + r.count - 1) / block - r.cached / block + 1) : 0;
    });
    // A thread's first vector, and the step from one of its vectors to the next, in rows and vectors of a row.
    const int row0 = threadIdx.x / per_row, column0 = threadIdx.x % per_row, row_step = threads / per_row, column_step = threads % per_row;
    const int blocks = prefix[batch], items = blocks * c.kv_heads * 2;
    // (Two places that take turns: one barrier per use is enough.)
    const auto block_largest = [&](uint32_t mine, int& turn) {
        mine = __reduce_max_sync(0xffffffffu, mine);
        if constexpr (kWarps > 1) {
            if (threadIdx.x % 32 == 0) largest_of[turn][threadIdx.x / 32] = mine;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mine = max(mine, largest_of[turn][w]);
            turn ^= 1;
        }
        return mine;
    };
    int turn = 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int head = item % c.kv_heads, pair = item / c.kv_heads, at = pair / 2;
        const bool is_value = pair % 2;
        const int row = row_of_item(prefix, batch, at);
        const NewRows r = new_rows(p, row);
        const int64_t index = r.cached / block + (at - prefix[row]), start = index * block;
        const int old = (int)max(r.cached - start, (int64_t)0);                         // positions of this block that stay
        const int end = (int)min(r.cached + r.count - start, (int64_t)block);           // positions that are filled then
        const int64_t stride = is_value ? p.value_stride : p.key_stride;
        const T* from = static_cast<const T*>(is_value ? p.values : p.keys);
        from += (r.begin + start + old - r.cached) * stride + head * c.head_dim;
        const int64_t row_head = (int64_t)row * c.kv_heads + head;
        uint8_t* codes = (is_value ? c.value_codes : c.key_codes) + (row_head * c.max_len + start) * c.head_dim;
        float* scale_at = (is_value ? c.value_scales : c.key_scales) + row_head * c.blocks + index;
        const float before = old > 0 ? *scale_at : 0.0f;

        // The new elements and their largest magnitude; where that is not finite, the largest finite one.
        V held[kVectors];
        const int rows = end - old;
        int i = row0, column = column0;
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            held[k].bits = make_uint4(0, 0, 0, 0);
            if (i < rows) held[k].bits = __ldg(reinterpret_cast<const uint4*>(from + (int64_t)i * stride) + column);
            i += row_step;
            column += column_step;
            if (column >= per_row) column -= per_row, ++i;
        }
        uint32_t largest = 0;
#pragma unroll
        for (int k = 0; k < kVectors; ++k) largest = V::larger(largest, held[k].bits);
        largest = block_largest(V::magnitude(largest), turn);
        if (largest >= 0x7f800000u) {  // (rare: out of memory once more, by all threads)
            largest = 0;
#pragma unroll 1
            for (int e = threadIdx.x; e < rows * c.head_dim; e += threads) {
                const uint32_t size = __float_as_uint(to_float(from[(int64_t)(e / c.head_dim) * stride + e % c.head_dim])) & 0x7fffffffu;
                if (size < 0x7f800000u) largest = max(largest, size);
            }
            largest = block_largest(largest, turn);
        }
        const float need = scale_of(__uint_as_float(largest));
        const float scale = old > 0 ? fmaxf(before, need) : need;
        const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0;  // (a cache filled by other means may have other scales)
        const float inverse = 1.0f / scale;
        uint8_t* to = codes + (int64_t)old * c.head_dim;
        if (power) {
            i = row0, column = column0;
            asm volatile("" : "+r"(i), "+r"(column));  // (counted once more: the registers are for the elements)
#pragma unroll
            for (int k = 0; k < kVectors; ++k) {
                if (i < rows) {
                    uint8_t* place = to + i * c.head_dim + column * V::elements;
                    const uint32_t first = held[k].codes(0, inverse);
                    if constexpr (V::elements == 4) *reinterpret_cast<uint32_t*>(place) = first;
                    else *reinterpret_cast<uint2*>(place) = make_uint2(first, held[k].codes(4, inverse));
                }
                i += row_step;
                column += column_step;
                if (column >= per_row) column -= per_row, ++i;
            }
        } else {  // (out of memory once more)
#pragma unroll 1
            for (int e = threadIdx.x; e < rows * c.head_dim; e += threads) {
                to[e] = (uint8_t)floats_to_codes(to_float(from[(int64_t)(e / c.head_dim) * stride + e % c.head_dim]) / scale, 0.0f);
            }
        }
        if (old > 0 && scale != before) {  // the codes that stay, in the new scale
            const float rate = before / scale;
            for (int v = threadIdx.x; v < old * c.head_dim / 4; v += threads) {
                const uint32_t four = reinterpret_cast<uint32_t*>(codes)[v];
                uint32_t made = 0;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t h = codes_to_halves(four >> (16 * half));
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
                    made |= floats_to_codes(x.x * rate, x.y * rate) << (16 * half);
                }
                reinterpret_cast<uint32_t*>(codes)[v] = made;
            }
        }
        if (threadIdx.x == 0) *scale_at = scale;  // (every thread has read it: it is this block's alone, and they have met since)
    }
}

template <class T, int threads>
cudaError_t launch_with(const StoreCacheParams& p, int sm_count, cudaStream_t stream) {
    const Cache8bitView& c = p.cache;
    // Blocks that the new positions can touch: every full one, and two more at the ends of each row.
    const int64_t touched = p.total / c.block + 2 * c.batch;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(touched * c.kv_heads * 2, (int64_t)sm_count * (512 / threads)));
    const size_t shared = (size_t)(c.batch + 1) * sizeof(int);
    store_cache_8bit_kernel<T, threads><<<grid, threads, shared, stream>>>(p);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch(const StoreCacheParams& p, int sm_count, cudaStream_t stream) {
    const int elements = p.cache.block * p.cache.head_dim;
    if (elements <= 32 * kHeld) return launch_with<T, 32>(p, sm_count, stream);
    if (elements <= 64 * kHeld) return launch_with<T, 64>(p, sm_count, stream);
    if (elements <= 128 * kHeld) return launch_with<T, 128>(p, sm_count, stream);
    return launch_with<T, 256>(p, sm_count, stream);
}

}  // namespace

cudaError_t launch_store_cache_8bit(const StoreCacheParams& p, int sm_count, cudaStream_t stream) {
    if (p.type == kFloat32) return launch<float>(p, sm_count, stream);
    if (p.type == kBfloat16) return launch<__nv_bfloat16>(p, sm_count, stream);
    return launch<__half>(p, sm_count, stream);
}

}  // namespace psx
