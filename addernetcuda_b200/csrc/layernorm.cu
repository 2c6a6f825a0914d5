// Layer norm over the last axis, forward and backward, with the sum of a residual stream before it.
//
//   h = round(x + residual), mean and var of h, rs = 1 / sqrt(var + eps), y = (h - mean) rs w + b
//   backward, with g = dy w and xh = (h - mean) rs:  dh = rs (g - mean(g) - xh mean(g xh)) [+ the gradient of h itself];
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// Bound by memory: x (and the residual) read, y (and h) written; h and dy (and dh) read, dx written.  A row is held in the registers of
// the threads that share it, so it is read once; a thread keeps its columns from row to row, and with them the weights and, in the
// backward pass, its sums of dw and db, which are added up over the CTAs by a second kernel, always in the same order.
//
// Measured (of a copy's rate): 8192x4096 bf16 with a residual stream forward 51 us (81 %), backward 50 us (82 %: some 5 us of it the second
// kernel); 16384x2048 fp32 48 us (86 %) and 68 us (90 %); 2000x20000 bf16 47 us (53 %: one CTA an SM goes over
// shared memory three times, with barriers between) and 106 us (35 %: long rows read h and dy once more for dw and db); 8192x1001 bf16, whose rows
// allow no vectors, 31 us and 41 us (32 and 24 %: two bytes at a time).
namespace adder {
namespace {
constexpr bool NORM_RMS = false;
}
}  // namespace adder
#include "norm.cuh"

using namespace adder;

extern "C" {

int adder_b200_layernorm_forward(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* h, float* mean,
                                 float* rstd, long long rows, long long d, long long x_stride, long long residual_stride, int dtype,
                                 int weight_dtype, float eps, void* stream) {
    const int st = ln_check(rows, d, dtype, weight_dtype);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!x || !y || (residual && !h) || !mean != !rstd) return ADDER_ERR_NULL_POINTER;
    if (!(eps >= 0.f) || x_stride < 0 || residual_stride < 0) return ADDER_ERR_BAD_SHAPE;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2, wsize = weight_dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!all_aligned({x, residual, y, h}, size) || !all_aligned({weight, bias}, wsize) || !all_aligned({mean, rstd}, 4)) return ADDER_ERR_ALIGNMENT;
    const LnFwd a{x, residual, weight, bias, y, h, mean, rstd, rows, x_stride, residual_stride, (int)d, eps, nullptr, 0};
    return norm_forward(a, dtype, weight_dtype, static_cast<cudaStream_t>(stream));
}

size_t adder_b200_layernorm_backward_workspace_bytes(long long rows, long long d) { return norm_backward_workspace_bytes(rows, d); }

int adder_b200_layernorm_backward(const void* dy, const void* dh, const void* h, const void* weight, const float* mean, const float* rstd,
                                  void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes, long long rows, long long d,
                                  long long h_stride, int dtype, int weight_dtype, void* stream) {
    const int st = ln_check(rows, d, dtype, weight_dtype);
    if (st != ADDER_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t wsize = weight_dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (rows == 0) {      // sums of nothing
        if ((dweight && cudaMemsetAsync(dweight, 0, d * wsize, s) != cudaSuccess) || (dbias && cudaMemsetAsync(dbias, 0, d * wsize, s) != cudaSuccess)) {
            (void)cudaGetLastError();
            return ADDER_ERR_CUDA;
        }
        return ADDER_OK;
    }
    if (!dy || !h || !mean || !rstd) return ADDER_ERR_NULL_POINTER;
    if (h_stride < 0) return ADDER_ERR_BAD_SHAPE;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!all_aligned({dy, dh, h, dx}, size) || !all_aligned({weight, dweight, dbias}, (unsigned)wsize) || !all_aligned({mean, rstd}, 4) || !aligned_to(workspace, 16))
        return ADDER_ERR_ALIGNMENT;
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (!sums && dx == nullptr) return ADDER_OK;
    if (sums && (workspace == nullptr || workspace_bytes < adder_b200_layernorm_backward_workspace_bytes(rows, d))) return ADDER_ERR_WORKSPACE;
    const LnBwd a{dy, dh, h, weight, mean, rstd, dx, rows, h_stride, (int)d};
    return norm_backward(a, dweight, dbias, workspace, dtype, weight_dtype, s);
}

}  // extern "C"
