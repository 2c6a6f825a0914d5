// Layer norm over the last axis, forward and backward, with the sum of a residual stream before it.
//
//   h = round(x + residual), mean and var of h, rs = 1 / sqrt(var + eps), y = (h - mean) rs w + b
//   backward, with g = dy w and xh = (h - mean) rs:  dh = rs (g - mean(g) - xh mean(g xh)) [+ the gradient of h itself];
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// Bound by memory: x (and the residual) read, y (and h) written; h and dy (and dh) read, dx written.  A row is held in the registers of
// the threads that share it, so it is read once; its variance is taken about its mean, in a second pass over the registers.
#include "kernels.h"
#include "elements.cuh"
#include <cooperative_groups.h>
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

namespace adder {
namespace {

namespace cg = cooperative_groups;

struct LnFwd {
    const void* x;
    const void* residual;      // may be null
    const void* w;             // may be null: 1
    const void* b;             // may be null: 0
    void* y;
    void* h;                   // with residual
    float* mean;               // may be null, with rstd
    float* rstd;
    long long rows, x_stride, r_stride;
    int d;
    float eps;
};

struct LnBwd {
    const void* dy;
    const void* dh;            // gradient of h, may be null
    const void* h;
    const void* w;
    const float* mean;
    const float* rstd;
    void* dx;
    long long rows, h_stride;
    int d;
};

template <class T, int N> __device__ __forceinline__ void load_some(const T* p, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = to_float(*p);
    } else {
        constexpr int V = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < N / V; ++i) {
            float v[V];
            Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p) + i), v);
#pragma unroll
            for (int j = 0; j < V; ++j) f[i * V + j] = v[j];
        }
    }
}
template <class T, int N> __device__ __forceinline__ void store_some(T* p, const float (&f)[N]) {
    if constexpr (N == 1) *p = from_float<T>(f[0]);
    else *reinterpret_cast<uint4*>(p) = Vec16<T>::pack(f);
}

// Sum over the G threads of a team; `part` is that team's own shared memory and is free again after the next barrier.
template <int G> __device__ __forceinline__ float team_sum(float v, float* part, int t) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if constexpr (G > 32) {
        if ((t & 31) == 0) part[t >> 5] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < G / 32; ++i) v += part[i];
    }
    return v;
}

template <int G> constexpr int LN_TEAMS = G >= 128 ? 1 : 128 / G;      // teams of a CTA

// A team of G threads a row, VEC consecutive elements at a time, NV times.
template <class T, class W, int G, int VEC, int NV>
__global__ void __launch_bounds__(G * LN_TEAMS<G>) ln_forward_kernel(const LnFwd a) {
    __shared__ float part[2][G / 32];
    const int t = threadIdx.x % G;
    const long long row = (long long)blockIdx.x * LN_TEAMS<G> + threadIdx.x / G;
    if (row >= a.rows) return;      // whole warps: a team of more is a CTA
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float f[NV][VEC];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.d) {
            load_some<T, VEC>(x + c, f[i]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[i][j] = 0.f;
        }
    }
    if (a.residual != nullptr) {
        const T* r = static_cast<const T*>(a.residual) + row * a.r_stride;
        T* h = static_cast<T*>(a.h) + row * (long long)a.d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VEC;
            if (c < a.d) {
                float g[VEC];
                load_some<T, VEC>(r + c, g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[i][j] = to_float(from_float<T>(f[i][j] + g[j]));      // the norm is taken of what is stored
                store_some<T, VEC>(h + c, f[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += f[i][j];
    const float mean = team_sum<G>(sum, part[0], t) / a.d;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * G + t) * VEC < a.d) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) sq += (f[i][j] - mean) * (f[i][j] - mean);
        }
    const float rs = 1.f / sqrtf(team_sum<G>(sq, part[1], t) / a.d + a.eps);
    if (t == 0 && a.mean != nullptr) { a.mean[row] = mean; a.rstd[row] = rs; }
    T* y = static_cast<T*>(a.y) + row * (long long)a.d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.d) {
            float w[VEC], b[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) { w[j] = 1.f; b[j] = 0.f; }
            if (a.w != nullptr) load_some<W, VEC>(static_cast<const W*>(a.w) + c, w);
            if (a.b != nullptr) load_some<W, VEC>(static_cast<const W*>(a.b) + c, b);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[i][j] = fmaf((f[i][j] - mean) * rs, w[j], b[j]);
            store_some<T, VEC>(y + c, f[i]);
        }
    }
}

template <class T, class W, int G, int VEC, int NV>
__global__ void __launch_bounds__(G * LN_TEAMS<G>) ln_dx_kernel(const LnBwd a) {
    __shared__ float part[2][G / 32];
    const int t = threadIdx.x % G;
    const long long row = (long long)blockIdx.x * LN_TEAMS<G> + threadIdx.x / G;
    if (row >= a.rows) return;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * (long long)a.d;
    const float mean = a.mean[row], rs = a.rstd[row];
    float g[NV][VEC], xh[NV][VEC];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.d) {
            float w[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[j] = 1.f;
            load_some<T, VEC>(h + c, xh[i]);
            load_some<T, VEC>(dy + c, g[i]);
            if (a.w != nullptr) load_some<W, VEC>(static_cast<const W*>(a.w) + c, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                g[i][j] *= w[j];
                xh[i][j] = (xh[i][j] - mean) * rs;
                s1 += g[i][j];
                s2 = fmaf(g[i][j], xh[i][j], s2);
            }
        }
    }
    s1 = team_sum<G>(s1, part[0], t) / a.d;
    s2 = team_sum<G>(s2, part[1], t) / a.d;
    T* dx = static_cast<T*>(a.dx) + row * (long long)a.d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.d) {
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = rs * (g[i][j] - s1 - xh[i][j] * s2);
            if (a.dh != nullptr) {
                float e[VEC];
                load_some<T, VEC>(static_cast<const T*>(a.dh) + row * (long long)a.d + c, e);
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] += e[j];
            }
            store_some<T, VEC>(dx + c, o);
        }
    }
}

// ------------------------------------------------------------------------------------------ rows too long for registers

constexpr int LN_LONG = 512;      // threads of each CTA of a cluster

// Sum over the CTAs of the cluster, in rank order.  `slot` is used once in a kernel.
__device__ __forceinline__ float cluster_sum(float v, float* part, float* slot, int t) {
    cg::cluster_group cluster = cg::this_cluster();
    v = team_sum<LN_LONG>(v, part, t);
    if (t == 0) *slot = v;
    cluster.sync();
    float all = 0.f;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) all += *cluster.map_shared_rank(slot, r);
    return all;
}

template <class T, class W> __global__ void __launch_bounds__(LN_LONG) ln_forward_long_kernel(const LnFwd a) {
    __shared__ float part[2][LN_LONG / 32], slot[2];
    const int t = threadIdx.x, parts = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const long long row = blockIdx.x / parts;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
    T* h = a.residual != nullptr ? static_cast<T*>(a.h) + row * (long long)a.d : nullptr;
    T* y = static_cast<T*>(a.y) + row * (long long)a.d;
    const int c0 = (int)((long long)a.d * rank / parts), c1 = (int)((long long)a.d * (rank + 1) / parts);
    const auto at = [&](int c) { return r == nullptr ? to_float(x[c]) : to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))); };
    float sum = 0.f, sq = 0.f;
    for (int c = c0 + t; c < c1; c += LN_LONG) sum += at(c);
    const float mean = cluster_sum(sum, part[0], slot, t) / a.d;
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float e = at(c) - mean;
        sq += e * e;
    }
    const float rs = 1.f / sqrtf(cluster_sum(sq, part[1], slot + 1, t) / a.d + a.eps);
    if (t == 0 && rank == 0 && a.mean != nullptr) { a.mean[row] = mean; a.rstd[row] = rs; }
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float v = at(c);
        if (h != nullptr) h[c] = from_float<T>(v);
        const float w = a.w != nullptr ? to_float(static_cast<const W*>(a.w)[c]) : 1.f, b = a.b != nullptr ? to_float(static_cast<const W*>(a.b)[c]) : 0.f;
        y[c] = from_float<T>(fmaf((v - mean) * rs, w, b));
    }
    cg::this_cluster().sync();      // no CTA leaves while its shared memory is read
}

template <class T, class W> __global__ void __launch_bounds__(LN_LONG) ln_dx_long_kernel(const LnBwd a) {
    __shared__ float part[2][LN_LONG / 32], slot[2];
    const int t = threadIdx.x, parts = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const long long row = blockIdx.x / parts;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * (long long)a.d;
    const T* dh = a.dh != nullptr ? static_cast<const T*>(a.dh) + row * (long long)a.d : nullptr;
    T* dx = static_cast<T*>(a.dx) + row * (long long)a.d;
    const float mean = a.mean[row], rs = a.rstd[row];
    const int c0 = (int)((long long)a.d * rank / parts), c1 = (int)((long long)a.d * (rank + 1) / parts);
    const auto weight = [&](int c) { return a.w != nullptr ? to_float(static_cast<const W*>(a.w)[c]) : 1.f; };
    float s1 = 0.f, s2 = 0.f;
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float g = to_float(dy[c]) * weight(c);
        s1 += g;
        s2 = fmaf(g, (to_float(h[c]) - mean) * rs, s2);
    }
    s1 = cluster_sum(s1, part[0], slot, t) / a.d;
    s2 = cluster_sum(s2, part[1], slot + 1, t) / a.d;
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float o = rs * (to_float(dy[c]) * weight(c) - s1 - (to_float(h[c]) - mean) * rs * s2);
        dx[c] = from_float<T>(dh != nullptr ? o + to_float(dh[c]) : o);
    }
    cg::this_cluster().sync();
}

// ------------------------------------------------------------------------------------------ gradients of weight and bias

constexpr int LN_COLS = 32, LN_LANES = 8;      // a CTA's columns, and the rows that it reads at once

// grid (column tiles, splits): part[split][2][d]
template <class T> __global__ void __launch_bounds__(LN_COLS * LN_LANES) ln_columns_kernel(const LnBwd a, float* part) {
    __shared__ float sw[LN_LANES][LN_COLS], sb[LN_LANES][LN_COLS];
    const int lane = threadIdx.x % LN_COLS, line = threadIdx.x / LN_COLS;
    const int c = blockIdx.x * LN_COLS + lane;
    float dw = 0.f, db = 0.f;
    if (c < a.d)
        for (long long row = (long long)blockIdx.y * LN_LANES + line; row < a.rows; row += (long long)gridDim.y * LN_LANES) {
            const float g = to_float(static_cast<const T*>(a.dy)[row * a.d + c]);
            dw = fmaf(g, (to_float(static_cast<const T*>(a.h)[row * a.h_stride + c]) - a.mean[row]) * a.rstd[row], dw);
            db += g;
        }
    sw[line][lane] = dw; sb[line][lane] = db;
    __syncthreads();
    if (line < 2 && c < a.d) {
        float s = 0.f;
        for (int i = 0; i < LN_LANES; ++i) s += line == 0 ? sw[i][lane] : sb[i][lane];
        part[((long long)blockIdx.y * 2 + line) * a.d + c] = s;
    }
}

template <class W> __global__ void __launch_bounds__(256) ln_columns_finish_kernel(const float* part, int splits, int d, W* dw, W* db) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= d) return;
    float w = 0.f, b = 0.f;
    for (int s = 0; s < splits; ++s) {
        w += part[((long long)s * 2) * d + c];
        b += part[((long long)s * 2 + 1) * d + c];
    }
    if (dw != nullptr) dw[c] = from_float<W>(w);
    if (db != nullptr) db[c] = from_float<W>(b);
}

// ------------------------------------------------------------------------------------------ host

int ln_splits(long long rows, int d) {
    const long long tiles = (d + LN_COLS - 1) / LN_COLS;
    long long splits = (8LL * sm_count() + tiles - 1) / tiles;
    splits = std::min(splits, (rows + LN_LANES - 1) / LN_LANES);
    return (int)std::max(1LL, std::min(splits, 1024LL));
}

template <class Args, class Kernel> int launch_long(const Args& a, Kernel kernel, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * 8));
    cfg.blockDim = dim3(LN_LONG);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 8; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
        (void)cudaGetLastError();
        return ADDER_ERR_CUDA;
    }
    count_launch();
    return ADDER_OK;
}

// A launch of the kernel whose registers hold a row of d elements, by f(G, VEC, NV) as integral constants; false: none does.
template <int N> using Int = std::integral_constant<int, N>;
template <int VE, class F> bool by_width(int d, bool vectors, F&& f) {
    if (vectors) {
        if (d <= 32 * VE) f(Int<32>(), Int<VE>(), Int<1>());
        else if (d <= 128 * VE) f(Int<32>(), Int<VE>(), Int<4>());
        else if (d <= 512 * VE) f(Int<128>(), Int<VE>(), Int<4>());
        else if (d <= 2048 * VE) f(Int<512>(), Int<VE>(), Int<4>());
        else return false;
    } else {
        if (d <= 128) f(Int<32>(), Int<1>(), Int<4>());
        else if (d <= 512) f(Int<32>(), Int<1>(), Int<16>());
        else if (d <= 2048) f(Int<128>(), Int<1>(), Int<16>());
        else if (d <= 8192) f(Int<512>(), Int<1>(), Int<16>());
        else return false;
    }
    return true;
}
template <class T, class F> int with_weight_type(int wtype, F&& f) {
    if (wtype == ADDER_TYPE_F32) return f(static_cast<float*>(nullptr));
    return f(static_cast<T*>(nullptr));
}

int ln_check(long long rows, long long d, int dtype, int wtype) {
    if (rows < 0 || d <= 0) return ADDER_ERR_BAD_SHAPE;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16 || (wtype != dtype && wtype != ADDER_TYPE_F32)) return ADDER_ERR_UNSUPPORTED;
    if (d > 2147483647LL - 65536 || rows > 2147483647LL / 8) return ADDER_ERR_UNSUPPORTED;
    return ADDER_OK;
}

bool all_aligned(std::initializer_list<const void*> ps, unsigned bytes) {
    for (const void* p : ps)
        if (!aligned_to(p, bytes)) return false;
    return true;
}

}  // namespace
}  // namespace adder

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
    const LnFwd a{x, residual, weight, bias, y, h, mean, rstd, rows, x_stride, residual_stride, (int)d, eps};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int VE = Vec16<T>::N;
        const bool vectors = d % VE == 0 && x_stride % VE == 0 && (!residual || residual_stride % VE == 0) &&
                             all_aligned({x, residual, weight, bias, y, h}, 16);
        return with_weight_type<T>(weight_dtype, [&](auto* wt) {
            using W = std::remove_pointer_t<decltype(wt)>;
            const bool held = by_width<VE>((int)d, vectors, [&](auto g, auto vec, auto nv) {
                constexpr int G = g, teams = LN_TEAMS<G>;
                ln_forward_kernel<T, W, G, vec, nv><<<(unsigned)((rows + teams - 1) / teams), G * teams, 0, s>>>(a);
            });
            return held ? launched() : launch_long(a, ln_forward_long_kernel<T, W>, s);
        });
    });
}

size_t adder_b200_layernorm_backward_workspace_bytes(long long rows, long long d) {
    if (rows <= 0 || d <= 0 || d > 2147483647LL - 65536) return 0;
    return (size_t)ln_splits(rows, (int)d) * 2 * d * sizeof(float);
}

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
    if (!all_aligned({dy, dh, h, dx}, size) || !all_aligned({weight, dweight, dbias}, (unsigned)wsize) || !all_aligned({mean, rstd, workspace}, 4))
        return ADDER_ERR_ALIGNMENT;
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (sums && (workspace == nullptr || workspace_bytes < adder_b200_layernorm_backward_workspace_bytes(rows, d))) return ADDER_ERR_WORKSPACE;
    const LnBwd a{dy, dh, h, weight, mean, rstd, dx, rows, h_stride, (int)d};
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int VE = Vec16<T>::N;
        const bool vectors = d % VE == 0 && h_stride % VE == 0 && all_aligned({dy, dh, h, weight, dx}, 16);
        return with_weight_type<T>(weight_dtype, [&](auto* wt) {
            using W = std::remove_pointer_t<decltype(wt)>;
            int status = ADDER_OK;
            if (dx != nullptr) {
                const bool held = by_width<VE>((int)d, vectors, [&](auto g, auto vec, auto nv) {
                    constexpr int G = g, teams = LN_TEAMS<G>;
                    ln_dx_kernel<T, W, G, vec, nv><<<(unsigned)((rows + teams - 1) / teams), G * teams, 0, s>>>(a);
                });
                status = held ? launched() : launch_long(a, ln_dx_long_kernel<T, W>, s);
            }
            if (status != ADDER_OK || !sums) return status;
            const int splits = ln_splits(rows, (int)d);
            float* part = static_cast<float*>(workspace);
            ln_columns_kernel<T><<<dim3((unsigned)((d + LN_COLS - 1) / LN_COLS), splits), LN_COLS * LN_LANES, 0, s>>>(a, part);
            ln_columns_finish_kernel<W><<<(unsigned)((d + 255) / 256), 256, 0, s>>>(part, splits, (int)d, static_cast<W*>(dweight), static_cast<W*>(dbias));
            return launched(2);
        });
    });
}

}  // extern "C"
