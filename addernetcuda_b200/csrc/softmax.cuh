// What the operators on rows of logits share: maxima that keep a NaN, and the exponential in base 2.
#pragma once
#include "elements.cuh"

namespace adder {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <class T> __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max_pair<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <> __device__ __forceinline__ uint32_t max_pair<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The largest of a vector's values, NaN if one is: as a word of its type, so that 16-bit values are compared in pairs.
template <class T> __device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    else return max_pair<T>(a, b);
}
template <class T> __device__ __forceinline__ float word_max(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(w);
    } else {
        const float2 p = unpack_pair<T>(w);
        return max_nan(p.x, p.y);
    }
}

}  // namespace adder
