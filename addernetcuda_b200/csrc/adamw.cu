// AdamW over all tensors of a model in one launch, states in 32 bits or as 8-bit codes.
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,  p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by memory: 28 bytes an element with fp32 parameters (p, g, m, v read, p, m, v written), 22 with 16-bit ones, 10 and 16 with 8-bit
// states.  A CTA takes one chunk of one tensor; which one it finds by bisection in a table that travels in the launch's
// parameters, so that nothing is copied to the device for it and a captured launch holds its own.
#include "kernels.h"
#include "elements.cuh"
#include <cmath>

namespace adder {
namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_CHUNK = AW_THREADS * 8;      // elements of one tensor that a CTA updates: 8 to a thread, one scale block to a warp
constexpr int AW_BLOCK = 256;                 // values that share a scale

using Tensor = adder_b200_adamw_tensor;

// 48 tensors fit in the 4 KB of parameters that every launch takes at full speed, 480 in the 32 KB that it takes at most.
template <int CAP> struct Table {
    Tensor t[CAP];
    int first[CAP + 1];      // first chunk of each tensor
    int count;
};

struct Hyper {
    float lr, b1, c1, b2, c2, eps, wd, ln_b1, ln_b2;      // c1 = 1 - b1, c2 = 1 - b2
    const float* lr_device;
    const float* grad_scale;
};

// Eight consecutive elements of a tensor, `valid` of them in it.
template <class T> __device__ __forceinline__ void load8(const T* p, int valid, float (&f)[8]) {
    constexpr int N = Vec16<T>::N;
    if (valid == 8 && aligned_to(p, 16)) {
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            float v[N];
            Vec16<T>::unpack(reinterpret_cast<const uint4*>(p)[i], v);
#pragma unroll
            for (int j = 0; j < N; ++j) f[i * N + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < valid ? to_float(p[i]) : 0.f;
    }
}
template <class T> __device__ __forceinline__ void store8(T* p, int valid, const float (&f)[8]) {
    constexpr int N = Vec16<T>::N;
    if (valid == 8 && aligned_to(p, 16)) {
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            float v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = f[i * N + j];
            reinterpret_cast<uint4*>(p)[i] = Vec16<T>::pack(v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = from_float<T>(f[i]);
    }
}
__device__ __forceinline__ uint2 load_codes(const unsigned char* p, int valid) {
    if (valid == 8 && aligned_to(p, 8)) return *reinterpret_cast<const uint2*>(p);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < valid) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(unsigned char* p, int valid, uint2 c) {
    if (valid == 8 && aligned_to(p, 8)) {
        *reinterpret_cast<uint2*>(p) = c;
        return;
    }
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < valid) p[i] = (unsigned char)(w[i >> 2] >> (8 * (i & 3)));
}

constexpr float TOP_M = 248.f, TOP_V = 63488.f, SMALLEST = 0x1p-100f;

// The magnitude of a code is the fp32 number with the code at bit 19 (a subnormal one where the exponent field is 0), times 2^127.
template <bool SIGNED> __device__ __forceinline__ float decode(uint32_t code, float scale) {
    const float mag = __fmul_rn(__uint_as_float((SIGNED ? code & 127u : code) << 19), 0x1p127f);
    return __fmul_rn(SIGNED && code >= 128u ? -mag : mag, scale);
}
template <bool SIGNED> __device__ __forceinline__ uint32_t encode(float x, float inv) {
    const uint32_t bits = __float_as_uint(__fmul_rn(__fmul_rn(fabsf(x), inv), 0x1p-127f));
    uint32_t code = min((bits + 0x3ffffu + ((bits >> 19) & 1u)) >> 19, SIGNED ? 127u : 255u);
    if (SIGNED) return x < 0.f ? code | 128u : code;
    return x > 0.f && inv > 0.f ? max(code, 1u) : code;
}

// Stores the warp's block of 256 values, eight to a lane.  Each operation rounds to fp32 by itself (no fused multiply-add), so that the
// codes are defined bit by bit.
template <bool SIGNED> __device__ __forceinline__ void store_block(unsigned char* codes, float* scale, int valid, const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);      // NaN above infinity above the rest
    float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, top));
    if (largest < SMALLEST) largest = 0.f;
    const float limit = SIGNED ? TOP_M : TOP_V;
    const float inv = largest > 0.f ? __fmul_rn(__frcp_rn(largest), limit) : 0.f;
    uint2 c = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.x |= encode<SIGNED>(x[i], inv) << (8 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.y |= encode<SIGNED>(x[i + 4], inv) << (8 * i);
    store_codes(codes, valid, c);
    if ((threadIdx.x & 31) == 0) *scale = __fmul_rn(largest, 1.f / limit);
}
template <bool SIGNED> __device__ __forceinline__ void load_block(const unsigned char* codes, const float* scale, int valid, float (&x)[8]) {
    const uint2 c = load_codes(codes, valid);
    const float sc = *scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = decode<SIGNED>((c.x >> (8 * i)) & 255u, sc);
        x[i + 4] = decode<SIGNED>((c.y >> (8 * i)) & 255u, sc);
    }
}

template <class T, int BITS, int CAP>
__global__ void __launch_bounds__(AW_THREADS) adamw_kernel(const __grid_constant__ Table<CAP> table, const __grid_constant__ Hyper h) {
    const int chunk = blockIdx.x;
    int lo = 0, hi = table.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    const Tensor& t = table.t[lo];
    const int step = t.step[0] + 1;
    // 1 - b^t through expm1, which keeps its digits where b^t is near 1
    const float lr = h.lr_device != nullptr ? *h.lr_device : h.lr;
    const float size = lr / -expm1f((float)step * h.ln_b1);
    const float root = rsqrtf(-expm1f((float)step * h.ln_b2));
    const float keep = 1.f - lr * h.wd;
    const float gs = h.grad_scale != nullptr ? *h.grad_scale : 1.f;

    const long long at = (long long)(chunk - table.first[lo]) * AW_CHUNK + threadIdx.x * 8;
    const long long left = t.n - at;
    const int valid = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    const long long block = at / AW_BLOCK;
    if (block * AW_BLOCK < t.n) {      // the same for all lanes of a warp
        float p[8], g[8], m[8], v[8];
        load8(static_cast<const T*>(t.param) + at, valid, p);
        load8(static_cast<const T*>(t.grad) + at, valid, g);
        if constexpr (BITS == 32) {
            load8(static_cast<const float*>(t.exp_avg) + at, valid, m);
            load8(static_cast<const float*>(t.exp_avg_sq) + at, valid, v);
        } else {
            load_block<true>(static_cast<const unsigned char*>(t.exp_avg) + at, t.exp_avg_scale + block, valid, m);
            load_block<false>(static_cast<const unsigned char*>(t.exp_avg_sq) + at, t.exp_avg_sq_scale + block, valid, v);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float gi = __fmul_rn(g[i], gs);
            m[i] = __fadd_rn(__fmul_rn(m[i], h.b1), __fmul_rn(gi, h.c1));
            v[i] = __fadd_rn(__fmul_rn(v[i], h.b2), __fmul_rn(__fmul_rn(gi, gi), h.c2));
            p[i] = p[i] * keep - size * __fdividef(m[i], fmaf(__fsqrt_rn(v[i]), root, h.eps));
        }
        store8(static_cast<T*>(t.param) + at, valid, p);
        if constexpr (BITS == 32) {
            store8(static_cast<float*>(t.exp_avg) + at, valid, m);
            store8(static_cast<float*>(t.exp_avg_sq) + at, valid, v);
        } else {
            store_block<true>(static_cast<unsigned char*>(t.exp_avg) + at, t.exp_avg_scale + block, valid, m);
            store_block<false>(static_cast<unsigned char*>(t.exp_avg_sq) + at, t.exp_avg_sq_scale + block, valid, v);
        }
    }
    // Every thread of every chunk has read the step count when the last chunk arrives: that one counts it up.
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(t.step + 1, 1) == table.first[lo + 1] - table.first[lo] - 1) {
            t.step[0] = step;
            t.step[1] = 0;
        }
    }
}

template <bool SIGNED>
__global__ void __launch_bounds__(AW_THREADS) adamw_values_kernel(const unsigned char* codes, const float* scales, float* values, long long n) {
    const long long at = ((long long)blockIdx.x * AW_THREADS + threadIdx.x) * 8;
    if (at >= n) return;
    const int valid = n - at >= 8 ? 8 : (int)(n - at);
    float x[8];
    load_block<SIGNED>(codes + at, scales + at / AW_BLOCK, valid, x);
    store8(values + at, valid, x);
}

template <class T, int CAP> int launch_table(const Table<CAP>& table, const Hyper& h, int bits, int chunks, cudaStream_t s) {
    if (bits == 32) adamw_kernel<T, 32, CAP><<<chunks, AW_THREADS, 0, s>>>(table, h);
    else adamw_kernel<T, 8, CAP><<<chunks, AW_THREADS, 0, s>>>(table, h);
    return launched();
}

// Launches over as many tensors from `tensors` on as a table takes; *next is the first that is left.
template <class T, int CAP> int launch_some(const Tensor* tensors, int count, int* next, const Hyper& h, int bits, cudaStream_t s) {
    Table<CAP> table;
    table.count = 0;
    long long chunks = 0;
    int i = *next;
    for (; i < count && table.count < CAP; ++i) {
        if (tensors[i].n == 0) continue;
        const long long more = (tensors[i].n + AW_CHUNK - 1) / AW_CHUNK;
        if (chunks + more > 2147483647LL) break;
        table.first[table.count] = (int)chunks;
        table.t[table.count++] = tensors[i];
        chunks += more;
    }
    *next = i;
    if (table.count == 0) return ADDER_OK;
    table.first[table.count] = (int)chunks;
    return launch_table<T, CAP>(table, h, bits, (int)chunks, s);
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_adamw_step(const adder_b200_adamw_tensor* tensors, int count, int dtype, int state_bits, double lr, const float* lr_device,
                          double beta1, double beta2, double eps, double weight_decay, const float* grad_scale, void* stream) {
    if (count < 0 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !std::isfinite(lr) ||
        !std::isfinite(weight_decay) || !std::isfinite(eps))
        return ADDER_ERR_BAD_SHAPE;
    if (state_bits != 32 && state_bits != 8) return ADDER_ERR_UNSUPPORTED;
    if (count == 0) return ADDER_OK;
    if (tensors == nullptr) return ADDER_ERR_NULL_POINTER;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    for (int i = 0; i < count; ++i) {
        const adder_b200_adamw_tensor& t = tensors[i];
        if (t.n < 0) return ADDER_ERR_BAD_SHAPE;
        if (t.n == 0) continue;
        if (t.n > (2147483647LL - 1) * AW_CHUNK) return ADDER_ERR_UNSUPPORTED;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || !t.step) return ADDER_ERR_NULL_POINTER;
        if (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return ADDER_ERR_NULL_POINTER;
        if (!aligned_to(t.param, size) || !aligned_to(t.grad, size) || !aligned_to(t.step, 4)) return ADDER_ERR_ALIGNMENT;
        if (state_bits == 32 ? !aligned_to(t.exp_avg, 4) || !aligned_to(t.exp_avg_sq, 4)
                             : !aligned_to(t.exp_avg_scale, 4) || !aligned_to(t.exp_avg_sq_scale, 4))
            return ADDER_ERR_ALIGNMENT;
    }
    Hyper h;
    h.lr = (float)lr; h.b1 = (float)beta1; h.c1 = (float)(1.0 - beta1); h.b2 = (float)beta2; h.c2 = (float)(1.0 - beta2);
    h.eps = (float)eps; h.wd = (float)weight_decay;
    h.ln_b1 = (float)std::log(beta1); h.ln_b2 = (float)std::log(beta2);      // -inf for 0: 1 - 0^t = 1
    h.lr_device = lr_device; h.grad_scale = grad_scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        for (int next = 0; next < count;) {
            const int st = count - next <= 48 ? launch_some<T, 48>(tensors, count, &next, h, state_bits, s)
                                              : launch_some<T, 480>(tensors, count, &next, h, state_bits, s);
            if (st != ADDER_OK) return st;
        }
        return (int)ADDER_OK;
    });
}

int adder_b200_adamw_state_values(const unsigned char* codes, const float* scales, int is_signed, float* values, long long n, void* stream) {
    if (n < 0) return ADDER_ERR_BAD_SHAPE;
    if (n == 0) return ADDER_OK;
    if (!codes || !scales || !values) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(scales, 4) || !aligned_to(values, 4)) return ADDER_ERR_ALIGNMENT;
    const long long grid = (n + AW_CHUNK - 1) / AW_CHUNK;
    if (grid > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (is_signed) adamw_values_kernel<true><<<(unsigned)grid, AW_THREADS, 0, s>>>(codes, scales, values, n);
    else adamw_values_kernel<false><<<(unsigned)grid, AW_THREADS, 0, s>>>(codes, scales, values, n);
    return launched();
}

}  // extern "C"
