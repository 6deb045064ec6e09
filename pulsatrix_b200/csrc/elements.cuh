// The element types that a call may name (psx_dtype), and 8-bit codes (e4m3: sign, 4 bits of exponent, 3 of fraction; no
// infinities, 0x7f and 0xff are NaN).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace psx {

enum ElementType { kFloat32 = 0, kBfloat16 = 1, kFloat16 = 2 };

__host__ __device__ constexpr int element_bytes(int type) { return type == kFloat32 ? 4 : 2; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Four consecutive elements as floats (one load of 16 or 8 bytes; p aligned to that).
template <class T>
__device__ __forceinline__ float4 load_four(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return __ldg(reinterpret_cast<const float4*>(p));
    } else {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
        T e[4];
        static_assert(sizeof(e) == sizeof(w));
        __builtin_memcpy(e, &w, sizeof(e));
        return make_float4(to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3]));
    }
}

// Two codes (the low 16 bits, lower byte first) as two halves: exact, every code but the two NaN is a half.
__device__ __forceinline__ uint32_t codes_to_halves(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
    return r;
}

// Four codes as two pairs of halves.
__device__ __forceinline__ void codes_to_halves(uint32_t four, uint32_t& low, uint32_t& high) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(low), "=r"(high) : "r"(four));
}

// Two floats, each rounded to the nearest code (ties to even), beyond the largest code to that; NaN stays NaN.
__device__ __forceinline__ uint32_t floats_to_codes(float low, float high) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace psx
