// Values in 8 bits: e4m3 codes that share an fp32 scale, a value being code * scale.
//
// A block's largest magnitude a gets the largest code: scale = a * (1 / 448), a value's code is e4m3(value * (1 / a * 448)), to nearest even, each
// operation rounded to fp32 (as the 8-bit states of the optimizer are stored).  Blocks whose largest magnitude is below 2^-100, where 448 / a
// nears the end of the range, are zeros.  A block with a NaN or an infinity stands for NaN as a whole.
#pragma once
#include "softmax.cuh"

namespace adder {

constexpr int E4M3_BLOCK = 128;         // columns (and rows of a weight) that share a scale
constexpr float E4M3_TOP = 448.f;

struct E4m3Scale {
    float scale, inverse;
};
__device__ __forceinline__ E4m3Scale e4m3_scale(float largest) {
    if (largest < 0x1p-100f) return {0.f, 0.f};
    return {__fmul_rn(largest, 1.f / E4M3_TOP), __fmul_rn(__frcp_rn(largest), E4M3_TOP)};
}
// Two codes, that of a in the low byte.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_word(float a, float b, float c, float d, float inverse) {
    return e4m3_pair(__fmul_rn(a, inverse), __fmul_rn(b, inverse)) | (e4m3_pair(__fmul_rn(c, inverse), __fmul_rn(d, inverse)) << 16);
}
__device__ __forceinline__ uint8_t e4m3_code(float a, float inverse) { return (uint8_t)e4m3_pair(__fmul_rn(a, inverse), 0.f); }

}  // namespace adder
