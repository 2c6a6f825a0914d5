// Element types of the operators that take more than fp32: loads, stores and conversions of one value or one vector.
// Everything is computed in fp32; a store to a 16-bit type rounds once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace adder {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// A pair of 16-bit values in one word.
template <class T> __device__ __forceinline__ float2 unpack_pair(uint32_t w);
template <> __device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack_pair<__half>(uint32_t w) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
template <class T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}

// What a 16-byte vector holds, as floats.
template <class T> struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[N]) {
        if constexpr (sizeof(T) == 4) {
            f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
        } else {
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = unpack_pair<T>(w[i]);
                f[2 * i] = v.x; f[2 * i + 1] = v.y;
            }
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[N]) {
        if constexpr (sizeof(T) == 4)
            return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        else
            return make_uint4(pack_pair<T>(f[0], f[1]), pack_pair<T>(f[2], f[3]), pack_pair<T>(f[4], f[5]), pack_pair<T>(f[6], f[7]));
    }
};

__host__ __device__ inline bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Calls f with a null pointer of the element type that an ADDER_TYPE_* code names.
template <class F> inline int with_type(int dtype, F&& f) {
    if (dtype == ADDER_TYPE_F32) return f(static_cast<float*>(nullptr));
    if (dtype == ADDER_TYPE_BF16) return f(static_cast<__nv_bfloat16*>(nullptr));
    if (dtype == ADDER_TYPE_F16) return f(static_cast<__half*>(nullptr));
    return ADDER_ERR_UNSUPPORTED;
}

}  // namespace adder
