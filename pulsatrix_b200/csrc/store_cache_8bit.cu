// New keys and values on their way into a cache held in 8 bits.
//
// A block of `block` positions of a (row, kv head) has one scale, a power of two: the least 2^e at which the block's largest
// magnitude, 448 * 2^e at most, has a code.  Codes are floating point themselves (e4m3), so a finer scale would buy no
// precision, and with powers of two nothing is rounded but the codes: values / scale is exact, and when a block that is
// partly filled has to grow its scale, the old codes times 2^(old - new) are exact too unless they fall below the smallest
// normal code.  A decoding step that adds one position at a time ends with what one call with all of them leaves, but for
// those.
//
// A block of threads takes (block of positions, kv head, keys or values): it holds its elements in registers between the
// maximum and the codes, so that the input is read once.  Bound by HBM for prompts, by latency for single positions.
#include "store_cache_8bit.cuh"

#include <algorithm>

#include "elements.cuh"
#include "row_prefix.cuh"

namespace psx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

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

template <class T, int vectors>
__global__ void __launch_bounds__(kThreads) store_cache_8bit_kernel(const __grid_constant__ StoreCacheParams p) {
    extern __shared__ int prefix[];
    __shared__ int carry[kWarps];
    __shared__ uint32_t largest_of[kWarps];
    const Cache8bitView& c = p.cache;
    const int batch = (int)c.batch, block = c.block, per_row = c.head_dim / 4;
    sum_of_rows(batch, prefix, carry, [&](int row) {
        const NewRows r = new_rows(p, row);
        if (p.row_status && blockIdx.x == 0) p.row_status[row] = r.status;
        return r.count ? (int)((r.cached + r.count - 1) / block - r.cached / block + 1) : 0;
    });
    const int64_t items = (int64_t)prefix[batch] * c.kv_heads * 2;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int head = (int)(item % c.kv_heads);
        const bool is_value = item / c.kv_heads % 2;
        const int at = (int)(item / c.kv_heads / 2);
        const int row = row_of_item(prefix, batch, at);
        const NewRows r = new_rows(p, row);
        const int64_t index = r.cached / block + (at - prefix[row]), start = index * block;
        const int old = (int)max(r.cached - start, (int64_t)0);                         // positions of this block that stay
        const int end = (int)min(r.cached + r.count - start, (int64_t)block);           // positions that are filled then
        const T* from = static_cast<const T*>(is_value ? p.values : p.keys);
        const int64_t stride = is_value ? p.value_stride : p.key_stride;
        from += (r.begin + start - r.cached) * stride + (int64_t)head * c.head_dim;     // (position 0 of the block, if it were new)
        const int64_t row_head = (int64_t)row * c.kv_heads + head;
        uint8_t* codes = (is_value ? c.value_codes : c.key_codes) + (row_head * c.max_len + start) * c.head_dim;
        float* scale_at = (is_value ? c.value_scales : c.key_scales) + row_head * c.blocks + index;
        const float before = old > 0 ? *scale_at : 0.0f;

        // The new elements, four at a time, and their largest finite magnitude.
        float4 held[vectors];
        uint32_t largest = 0;
        const int first = old * per_row, last = end * per_row;  // vectors of four
#pragma unroll
        for (int i = 0; i < vectors; ++i) {
            const int v = first + i * kThreads + (int)threadIdx.x;
            held[i] = make_float4(0, 0, 0, 0);
            if (v < last) held[i] = load_four(from + (int64_t)(v / per_row) * stride + v % per_row * 4);
        }
#pragma unroll
        for (int i = 0; i < vectors; ++i) {
            for (const float x : {held[i].x, held[i].y, held[i].z, held[i].w}) {
                const uint32_t size = __float_as_uint(x) & 0x7fffffffu;
                if (size < 0x7f800000u) largest = max(largest, size);
            }
        }
        largest = __reduce_max_sync(0xffffffffu, largest);
        if (threadIdx.x % 32 == 0) largest_of[threadIdx.x / 32] = largest;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) largest = max(largest, largest_of[w]);
        const float need = scale_of(__uint_as_float(largest));
        const float scale = old > 0 ? fmaxf(before, need) : need;
        const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0;  // (a cache filled by other means may have other scales)
        const float inverse = 1.0f / scale;
#pragma unroll
        for (int i = 0; i < vectors; ++i) {
            const int v = first + i * kThreads + (int)threadIdx.x;
            if (v >= last) continue;
            float4 x = held[i];
            if (power) x = make_float4(x.x * inverse, x.y * inverse, x.z * inverse, x.w * inverse);
            else x = make_float4(x.x / scale, x.y / scale, x.z / scale, x.w / scale);
            reinterpret_cast<uint32_t*>(codes)[v] = floats_to_codes(x.x, x.y) | floats_to_codes(x.z, x.w) << 16;
        }
        if (old > 0 && scale != before) {  // the codes that stay, in the new scale
            const float rate = before / scale;
            for (int v = threadIdx.x; v < first; v += kThreads) {
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
        if (threadIdx.x == 0) *scale_at = scale;
        __syncthreads();  // (largest_of is free for the next item; every thread has read the scale)
    }
}

template <class T>
cudaError_t launch(const StoreCacheParams& p, int sm_count, cudaStream_t stream) {
    const Cache8bitView& c = p.cache;
    // Blocks that the new positions can touch: every full one, and two more at the ends of each row.
    const int64_t touched = p.total / c.block + 2 * c.batch;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(touched * c.kv_heads * 2, (int64_t)sm_count * 8));
    const size_t shared = (size_t)(c.batch + 1) * sizeof(int);
    const int vectors = (c.block * c.head_dim / 4 + kThreads - 1) / kThreads;
    if (vectors <= 4) store_cache_8bit_kernel<T, 4><<<grid, kThreads, shared, stream>>>(p);
    else if (vectors <= 8) store_cache_8bit_kernel<T, 8><<<grid, kThreads, shared, stream>>>(p);
    else store_cache_8bit_kernel<T, 16><<<grid, kThreads, shared, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_store_cache_8bit(const StoreCacheParams& p, int sm_count, cudaStream_t stream) {
    if (p.type == kFloat32) return launch<float>(p, sm_count, stream);
    if (p.type == kBfloat16) return launch<__nv_bfloat16>(p, sm_count, stream);
    return launch<__half>(p, sm_count, stream);
}

}  // namespace psx
