// RMS norm over the last axis, forward and backward, with the sum of a residual stream before it, and with its output in 8 bits.
//
//   h = round(x + residual), rs = 1 / sqrt(mean(h^2) + eps), y = h rs w
//   backward, with g = dy w and xh = h rs:  dh = rs (g - xh mean(g xh)) [+ the gradient of h itself];  dw = sum over rows of dy xh
//   in 8 bits:  of each row and 128 columns a = max |y|, scale = a / 448, codes = e4m3(y 448 / a)
//
// Kernels of layer norm without its mean and bias (norm.cuh).  With the output in 8 bits a block of 128 columns lies with 16 (32, fp32)
// neighbouring lanes, which find its largest value by shuffles, so y is never written in 16 bits.
//
// Bound by memory, as layer norm is: 8192x4096 bf16 with a residual stream forward 39 us (the last rows still in L2), backward 45, both in turn 94 (87 % of
// a copy's rate); 8192x8192 bf16 with a stream to 8 bits 81 us (89 %).  2051x1001 fp32, rows that are no vectors, 6.2 and 14 us.  One row of 2048
// takes 4.3 us, a launch and two barriers.
namespace adder {
namespace {
constexpr bool NORM_RMS = true;
}
}  // namespace adder
#include "norm.cuh"

namespace adder {
namespace {

constexpr int RMS_ANY = 512;

// y in 8 bits of rows that are no whole vectors, or longer than registers hold: a CTA reads its row twice, the second time from L2.
template <class T, class W> __global__ void __launch_bounds__(RMS_ANY) rms_eight_any_kernel(const LnFwd a) {
    __shared__ float part[RMS_ANY / 32];
    const int t = threadIdx.x, lane = t & 31;
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
    T* h = a.residual != nullptr ? static_cast<T*>(a.h) + row * (long long)a.d : nullptr;
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride;
    const int blocks = (a.d + E4M3_BLOCK - 1) / E4M3_BLOCK;
    const auto at = [&](int c) { return r == nullptr ? to_float(x[c]) : to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))); };
    float sq = 0.f;
#pragma unroll 4
    for (int c = t; c < a.d; c += RMS_ANY) {
        const float v = at(c);
        if (h != nullptr) h[c] = from_float<T>(v);
        sq = fmaf(v, v, sq);
    }
    const float rs = inverse_root(team_sum<RMS_ANY>(sq, part, t) / a.d + a.eps);
    for (int b = t >> 5; b < blocks; b += RMS_ANY / 32) {
        float v[4], largest = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = b * E4M3_BLOCK + 32 * j + lane;
            v[j] = c < a.d ? at(c) * rs * (a.w != nullptr ? to_float(static_cast<const W*>(a.w)[c]) : 1.f) : 0.f;
            largest = max_nan(largest, fabsf(v[j]));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, off));
        const E4m3Scale s = e4m3_scale(largest);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = b * E4M3_BLOCK + 32 * j + lane;
            if (c < a.d) y[c] = e4m3_code(v[j], s.inverse);
        }
        if (lane == 0) a.scales[row * blocks + b] = s.scale;
    }
}

// f(shape) for the ring shape that holds a row of d elements, at most LN_HELD.
template <class T, class W, class F> int with_ring(int d, F&& f) {
    constexpr int VE = Vec16<T>::N, NV = 16 / VE, STAGES = NV == 2 ? 3 : 2;
    if (d <= 32 * VE) return f(LnShape<T, W, 32, VE, 1, 3, false>());
    if (d <= 512) return f(LnShape<T, W, 32, VE, NV, STAGES, false>());
    if (d <= 1024) return f(LnShape<T, W, 64, VE, NV, STAGES, false>());
    if (d <= 2048) return f(LnShape<T, W, 128, VE, NV, STAGES, false>());
    if (d <= 4096) return f(LnShape<T, W, 256, VE, NV, STAGES, false>());
    return f(LnShape<T, W, 512, VE, NV, 2, false>());
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_rmsnorm_forward(const void* x, const void* residual, const void* weight, void* y, void* h, float* rstd, long long rows, long long d,
                               long long x_stride, long long residual_stride, int dtype, int weight_dtype, float eps, void* stream) {
    const int st = ln_check(rows, d, dtype, weight_dtype);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!x || !y || (residual && !h)) return ADDER_ERR_NULL_POINTER;
    if (!(eps >= 0.f) || x_stride < 0 || residual_stride < 0) return ADDER_ERR_BAD_SHAPE;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2, wsize = weight_dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!all_aligned({x, residual, y, h}, size) || !aligned_to(weight, wsize) || !aligned_to(rstd, 4)) return ADDER_ERR_ALIGNMENT;
    const LnFwd a{x, residual, weight, nullptr, y, h, nullptr, rstd, rows, x_stride, residual_stride, (int)d, eps, nullptr, 0};
    return norm_forward(a, dtype, weight_dtype, static_cast<cudaStream_t>(stream));
}

int adder_b200_rmsnorm_forward_8bit(const void* x, const void* residual, const void* weight, void* values, float* scales, void* h, long long rows,
                                    long long d, long long x_stride, long long residual_stride, long long values_stride, int dtype,
                                    int weight_dtype, float eps, void* stream) {
    const int st = ln_check(rows, d, dtype, weight_dtype);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!x || !values || !scales || (residual && !h)) return ADDER_ERR_NULL_POINTER;
    if (!(eps >= 0.f) || x_stride < 0 || residual_stride < 0 || values_stride < d) return ADDER_ERR_BAD_SHAPE;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2, wsize = weight_dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!all_aligned({x, residual, h}, size) || !aligned_to(weight, wsize) || !aligned_to(scales, 4)) return ADDER_ERR_ALIGNMENT;
    const LnFwd a{x, residual, weight, nullptr, values, h, nullptr, nullptr, rows, x_stride, residual_stride, (int)d, eps, scales, values_stride};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int VE = Vec16<T>::N;
        const bool vectors = ln_vector<T>((int)d, {x_stride, residual ? residual_stride : 0}, {x, residual, h}, {weight}, wsize) == VE &&
                             values_stride % VE == 0 && aligned_to(values, VE);
        return with_weight_type<T>(weight_dtype, [&](auto* wt) {
            using W = std::remove_pointer_t<decltype(wt)>;
            if (vectors && d <= LN_HELD) return with_ring<T, W>((int)d, [&](auto shape) { return launch_forward<decltype(shape), true>(a, 1, s); });
            rms_eight_any_kernel<T, W><<<(unsigned)rows, RMS_ANY, 0, s>>>(a);
            return launched();
        });
    });
}

size_t adder_b200_rmsnorm_backward_workspace_bytes(long long rows, long long d) { return norm_backward_workspace_bytes(rows, d); }

int adder_b200_rmsnorm_backward(const void* dy, const void* dh, const void* h, const void* weight, const float* rstd, void* dx, void* dweight,
                                void* workspace, size_t workspace_bytes, long long rows, long long d, long long h_stride, int dtype, int weight_dtype,
                                void* stream) {
    const int st = ln_check(rows, d, dtype, weight_dtype);
    if (st != ADDER_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2, wsize = weight_dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (rows == 0) {      // a sum of nothing
        if (dweight && cudaMemsetAsync(dweight, 0, d * wsize, s) != cudaSuccess) {
            (void)cudaGetLastError();
            return ADDER_ERR_CUDA;
        }
        return ADDER_OK;
    }
    if (!dy || !h || !rstd) return ADDER_ERR_NULL_POINTER;
    if (h_stride < 0) return ADDER_ERR_BAD_SHAPE;
    if (!all_aligned({dy, dh, h, dx}, size) || !all_aligned({weight, dweight}, wsize) || !aligned_to(rstd, 4) || !aligned_to(workspace, 16))
        return ADDER_ERR_ALIGNMENT;
    if (dweight == nullptr && dx == nullptr) return ADDER_OK;
    if (dweight != nullptr && (workspace == nullptr || workspace_bytes < norm_backward_workspace_bytes(rows, d))) return ADDER_ERR_WORKSPACE;
    const LnBwd a{dy, dh, h, weight, nullptr, rstd, dx, rows, h_stride, (int)d};
    return norm_backward(a, dweight, nullptr, workspace, dtype, weight_dtype, s);
}

}  // extern "C"
