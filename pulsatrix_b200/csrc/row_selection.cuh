// What the kernels share that look for the largest logits of rows and sum their exponentials (beam_select.cu, token_log_probs.cu; warp_bound is beam_select's).
#pragma once

#include <stdint.h>

#include "elements.cuh"

namespace psx {

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

// A number that at least `keep` of the numbers of a block of `warps` warps reach, given every thread's largest (-inf where it has none): the
// smallest of the warps' n-th largest maxima, n = ceil(keep / warps).  Lanes of equal maxima leave together, which can only lower it.
template <int warps>
__device__ __forceinline__ uint32_t warp_bound(float largest, int keep, uint32_t* top) {
    uint32_t key = ordered(largest), bound = 0;
    for (int n = (keep + warps - 1) / warps; n > 0; --n) {
        bound = __reduce_max_sync(0xffffffffu, key);
        if (top) *top = bound, top = nullptr;
        key = key == bound ? 0u : key;
        if (bound <= ordered(kNone)) return 0;
    }
    return bound;
}

template <int warps>
__device__ __forceinline__ uint64_t block_max(uint64_t key, uint64_t* shared) {
    for (int step = 16; step > 0; step /= 2) key = max(key, __shfl_xor_sync(0xffffffffu, key, step));
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = key;
    __syncthreads();
    for (int w = 0; w < warps; ++w) key = max(key, shared[w]);
    __syncthreads();
    return key;
}

// {a, b} + {x, x}, {a, b} * {x, x} and {a, b} * {x, x} + {c, c}, each rounded as alone.
__device__ __forceinline__ float2 add_pair(float2 a, float2 x) {
    float2 r;
    asm("{\n\t.reg .b64 a, x, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tadd.rn.f32x2 r, a, x;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(x.x), "f"(x.y));
    return r;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 x) {
    float2 r;
    asm("{\n\t.reg .b64 a, x, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmul.rn.f32x2 r, a, x;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(x.x), "f"(x.y));
    return r;
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 x, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, x, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 r, a, x, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(x.x), "f"(x.y), "f"(c.x), "f"(c.y));
    return r;
}

// 2 atanh(z) by its power series up to z^15 (for |z| < 0.1716 what is left out is below 2^-44 of it).
__device__ __forceinline__ double twice_atanh(double z) {
    const double w = z * z;
    double series = 1.0 / 15.0;
#pragma unroll
    for (int n = 13; n > 0; n -= 2) series = fma(series, w, 1.0 / n);
    return 2.0 * z * series;
}

// The logarithm of a sum, in double precision: x = 2^e f with f between sqrt(1/2) and sqrt(2), log f = 2 atanh(z) with
// z = (f - 1) / (f + 1).  A sum just above 1, a token that is nearly certain, has its own logarithm, which a float's fraction would lose
// below 2^-24.
__device__ __forceinline__ double log_of(double x) {
    const int high = __double2hiint(x);
    int exponent = (high >> 20) - 1023;
    double f = __hiloint2double((high & 0xfffff) | 0x3ff00000, __double2loint(x));
    if (f > 1.4142135623730951) f *= 0.5, ++exponent;
    return fma((double)exponent, 0.6931471805599453, twice_atanh((f - 1.0) / (f + 1.0)));
}

// log(1 + r) for r >= 0, however small.
__device__ __forceinline__ double log_of_one_and(double r) { return r < 0.4 ? twice_atanh(r / (2.0 + r)) : log_of(1.0 + r); }

}  // namespace psx
