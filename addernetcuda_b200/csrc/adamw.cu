// AdamW over all tensors of a model in one launch, states in 32 bits or as 8-bit codes.
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,  p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by memory: 28 bytes an element with fp32 parameters (p, g, m, v read, p, m, v written), 22 with 16-bit ones, 10 and 16 with 8-bit
// states.  A CTA takes one chunk of one tensor; which one it finds by bisection in a table that travels in the launch's
// parameters, so that nothing is copied to the device for it and a captured launch holds its own.  A warp's next tiles are on their way
// through shared memory while it computes.
//
// Measured (of a copy's rate): 101 M fp32 elements 418 us and 48 M bf16 ones 160 us (all of it), 25 M fp32 ones 109 us (98 %); 201 M bf16 with 8-bit
// states 390 us (79 %), where instructions bound it as well: some 490 of a warp for 256 elements, issued in 84 % of the cycles (50 M elements).
#include "kernels.h"
#include "elements.cuh"
#include <cmath>

namespace adder {
namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_TILE = AW_THREADS * 8;       // elements that a CTA takes at once: 8 to a thread, one scale block to a warp
constexpr int AW_BLOCK = 256;                 // values that share a scale

using Tensor = adder_b200_adamw_tensor;

// 48 tensors fit in 4 KB of launch parameters, 480 in the 32 KB that there may be.  The host takes longer to launch larger ones (9.1, 9.9 and 12.5
// us a call with 48, 176 and 480), the kernel itself does not.
template <int CAP> struct Table {
    Tensor t[CAP];
    int first[CAP + 1];      // first chunk of each tensor
    int count, tiles;        // tiles of a chunk
};

struct Hyper {
    float lr, b1, c1, b2, c2, eps, wd, ln_b1, ln_b2;      // c1 = 1 - b1, c2 = 1 - b2
    const float* lr_device;
    const float* grad_scale;
};

// Eight consecutive elements of a tensor as they lie in memory, `valid` of them in it (zeros in place of the others).
template <class T> struct Raw8 {
    static constexpr int Q = sizeof(T) / 2;      // 16-byte words
    uint4 q[Q];
    // all eight, from shared memory
    __device__ __forceinline__ void read(uint32_t at) {
#pragma unroll
        for (int i = 0; i < Q; ++i)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[i].x), "=r"(q[i].y), "=r"(q[i].z), "=r"(q[i].w) : "r"(at + 16 * i) : "memory");
    }
    __device__ __forceinline__ void load(const T* p, int valid) {
        uint32_t w[4 * Q];
#pragma unroll
        for (int i = 0; i < 4 * Q; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(p[i]);
                else w[i / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i & 1));
            }
#pragma unroll
        for (int i = 0; i < Q; ++i) q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    // as four pairs of fp32
    __device__ __forceinline__ void pairs(uint64_t (&f)[4]) const {
        if constexpr (sizeof(T) == 4) {
            f[0] = pack2(__uint_as_float(q[0].x), __uint_as_float(q[0].y)); f[1] = pack2(__uint_as_float(q[0].z), __uint_as_float(q[0].w));
            f[2] = pack2(__uint_as_float(q[Q - 1].x), __uint_as_float(q[Q - 1].y)); f[3] = pack2(__uint_as_float(q[Q - 1].z), __uint_as_float(q[Q - 1].w));
        } else {
            const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = unpack_pair<T>(w[i]);
                f[i] = pack2(v.x, v.y);
            }
        }
    }
};
template <bool WHOLE, class T> __device__ __forceinline__ void store8(T* p, int valid, const uint64_t (&pairs)[4]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2(pairs[i], f[2 * i], f[2 * i + 1]);
    if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = from_float<T>(f[i]);
    } else if constexpr (sizeof(T) == 4) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]) : "memory");
    } else {
        *reinterpret_cast<uint4*>(p) = Vec16<T>::pack(f);
    }
}
template <bool WHOLE> __device__ __forceinline__ uint2 load_codes(const unsigned char* p, int valid) {
    if constexpr (WHOLE) return *reinterpret_cast<const uint2*>(p);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < valid) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
template <bool WHOLE> __device__ __forceinline__ void store_codes(unsigned char* p, int valid, uint2 c) {
    if constexpr (WHOLE) {
        *reinterpret_cast<uint2*>(p) = c;
        return;
    }
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < valid) p[i] = (unsigned char)(w[i >> 2] >> (8 * (i & 3)));
}

constexpr float TOP_M = 248.f, TOP_V = 63488.f, SMALLEST = 0x1p-100f;
__device__ __forceinline__ uint64_t twice(float v) { return pack2(v, v); }

// The magnitude of a code is the fp32 number with the code at bit 19 (a subnormal one where the exponent field is 0), times 2^127; a sign at bit
// 7 of the code goes to bit 31.  Eight codes, as pairs.  What bounds the 8-bit step beside memory is the integer pipe, half as wide as the
// one that multiplies: shifts are products here.
template <bool SIGNED> __device__ __forceinline__ float code_bits(uint32_t word, int i) {
    const uint32_t at19 = __byte_perm(word, 0, 0x4044 | (i << 8)) * 8u;
    if (!SIGNED) return __uint_as_float(at19);
    return __uint_as_float((at19 & (1u << 26)) * 31u + at19);      // 2^26 becomes 2^31
}
template <bool SIGNED> __device__ __forceinline__ void decode(uint2 c, float scale, uint64_t (&x)[4]) {
    const uint64_t up = twice(0x1p127f), sc = twice(scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t word = i < 2 ? c.x : c.y;
        x[i] = mul2(mul2(pack2(code_bits<SIGNED>(word, 2 * (i & 1)), code_bits<SIGNED>(word, 2 * (i & 1) + 1)), up), sc);
    }
}

// Code of a magnitude that has been scaled to the code's range and by 2^-127: rounded to nearest even at bit 19, moved to the top byte.
__device__ __forceinline__ uint32_t round_to_code(float scaled) {
    const uint32_t bits = __float_as_uint(scaled);
    return (bits + 0x3ffffu + ((bits >> 19) & 1u)) * 32u;
}
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// Stores the warp's block of 256 values, eight to a lane.  Each operation rounds to fp32 by itself, so that the codes are defined bit by
// bit.
template <bool SIGNED, bool WHOLE> __device__ __forceinline__ void store_block(unsigned char* codes, float* scale, int valid, const uint64_t (&x)[4]) {
    float f[8], top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2(x[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(f[i])));
    float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));      // NaN above infinity above the rest
    if (largest < SMALLEST) largest = 0.f;
    const float limit = SIGNED ? TOP_M : TOP_V;
    const float inv = largest > 0.f ? __fmul_rn(__frcp_rn(largest), limit) : 0.f;
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2(mul2(mul2(x[i], twice(inv)), twice(0x1p-127f)), a, b);
        r[2 * i] = round_to_code(a);
        r[2 * i + 1] = round_to_code(b);
    }
    uint32_t c[2] = {top_bytes(r[0], r[1], r[2], r[3]), top_bytes(r[4], r[5], r[6], r[7])};
    if (largest == 0.f) c[0] = c[1] = 0;
    if constexpr (SIGNED) {      // a negative value keeps its sign where it rounds to 0; -0, which is none, loses it in the sum with 0
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(add2(x[i], 0), f[2 * i], f[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t signs = top_bytes(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
            c[i] = (c[i] & 0x7f7f7f7fu) | (signs & 0x80808080u);
        }
    } else if (largest > 0.f) {      // a value above 0 has code 1 at least
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if ((c[i] - 0x01010101u) & ~c[i] & 0x80808080u) {      // a byte of 0 among the four
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (((c[i] >> (8 * j)) & 255u) == 0 && f[4 * i + j] > 0.f) c[i] |= 1u << (8 * j);
            }
    }
    store_codes<WHOLE>(codes, valid, make_uint2(c[0], c[1]));
    if ((threadIdx.x & 31) == 0) *scale = __fmul_rn(largest, 1.f / limit);
}

// Approximate to 2^-23 or so, like the root below.  Its operand, root(v) + eps, is no subnormal number: the root of the smallest v is 2^-74.5,
// and an eps between 0 and 2^-126 is refused.
__device__ __forceinline__ float reciprocal_of(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// FLUSH: 0 below 2^-126.
template <bool FLUSH> __device__ __forceinline__ float root_of(float x) {
    float r;
    if constexpr (FLUSH) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    else asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A thread's places in the tensors, and what it reads there.
template <class T, int BITS> struct Place {
    T* p;
    const T* g;
    float *m, *v;
    __device__ __forceinline__ Place(const Tensor& t, long long at)
        : p(static_cast<T*>(t.param) + at), g(static_cast<const T*>(t.grad) + at), m(static_cast<float*>(t.exp_avg) + at), v(static_cast<float*>(t.exp_avg_sq) + at) {}
    __device__ __forceinline__ void advance() { p += AW_TILE; g += AW_TILE; m += AW_TILE; v += AW_TILE; }
    __device__ __forceinline__ bool whole() const { return aligned_to(p, 8 * sizeof(T)) && aligned_to(g, 4) && aligned_to(m, 32) && aligned_to(v, 32); }
};
template <class T> struct Place<T, 8> {
    T* p;
    const T* g;
    unsigned char *m, *v;
    float *sm, *sv;
    __device__ __forceinline__ Place(const Tensor& t, long long at)
        : p(static_cast<T*>(t.param) + at), g(static_cast<const T*>(t.grad) + at), m(static_cast<unsigned char*>(t.exp_avg) + at),
          v(static_cast<unsigned char*>(t.exp_avg_sq) + at), sm(t.exp_avg_scale + at / AW_BLOCK), sv(t.exp_avg_sq_scale + at / AW_BLOCK) {}
    __device__ __forceinline__ void advance() {
        p += AW_TILE; g += AW_TILE; m += AW_TILE; v += AW_TILE;
        sm += AW_TILE / AW_BLOCK; sv += AW_TILE / AW_BLOCK;
    }
    __device__ __forceinline__ bool whole() const { return aligned_to(p, 8 * sizeof(T)) && aligned_to(g, 4) && aligned_to(m, 8) && aligned_to(v, 8); }
};
// A warp's 256 elements of each tensor on their way through shared memory, STAGES tiles deep.  Lanes copy consecutive 16-byte words, so what
// a lane reads may be another's copy: the warp waits for its copies together.  Offsets in a stage, in bytes.
template <class T, int BITS> struct Ring {
    static constexpr int E = AW_BLOCK * sizeof(T), F = BITS == 32 ? AW_BLOCK * 4 : AW_BLOCK;
    static constexpr int P = 0, G = E, M = 2 * E, V = 2 * E + F, S = 2 * E + 2 * F, STAGE = S + (BITS == 8 ? 16 : 0);
    static constexpr int STAGES = BITS == 8 ? 4 : sizeof(T) == 2 ? 3 : 2;
    static constexpr int WARP = STAGES * STAGE, BYTES = AW_THREADS / 32 * WARP;

    template <int N> static __device__ __forceinline__ void copy(uint32_t to, const void* from, int lane) {      // N bytes
        const char* p = static_cast<const char*>(from);
        if constexpr (N >= 512) {
#pragma unroll
            for (int i = 0; i < N / 512; ++i)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + 512 * i + 16 * lane), "l"(p + 512 * i + 16 * lane) : "memory");
        } else {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to + 8 * lane), "l"(p + 8 * lane) : "memory");
        }
    }
    // The same in words of 4 bytes, for gradients that lie one behind another in a bucket.
    static __device__ __forceinline__ void copy_words(uint32_t to, const void* from, int lane) {
#pragma unroll
        for (int i = 0; i < E / 128; ++i)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to + 128 * i + 4 * lane), "l"(static_cast<const char*>(from) + 128 * i + 4 * lane) : "memory");
    }
    // `at` is of the warp's first element
    static __device__ __forceinline__ void fill(uint32_t stage, const Place<T, BITS>& at, int tile, int lane) {
        const int o = tile * AW_TILE;
        copy<E>(stage + P, at.p + o, lane);
        if (aligned_to(at.g, 16)) copy<E>(stage + G, at.g + o, lane);      // the same for all of a tensor
        else copy_words(stage + G, at.g + o, lane);
        copy<F>(stage + M, at.m + o, lane);
        copy<F>(stage + V, at.v + o, lane);
        if constexpr (BITS == 8) {
            const int b = tile * (AW_TILE / AW_BLOCK);
            if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(stage + S + 4 * lane), "l"((lane == 0 ? at.sm : at.sv) + b) : "memory");
        }
    }
};

template <class T, int BITS> struct Tile {
    Raw8<T> p, g;
    Raw8<float> m, v;
    __device__ __forceinline__ void load(const Place<T, BITS>& at, int valid) {
        p.load(at.p, valid); g.load(at.g, valid); m.load(at.m, valid); v.load(at.v, valid);
    }
    __device__ __forceinline__ void read(uint32_t stage, int lane) {
        using R = Ring<T, BITS>;
        p.read(stage + R::P + lane * 8 * sizeof(T)); g.read(stage + R::G + lane * 8 * sizeof(T));
        m.read(stage + R::M + lane * 32); v.read(stage + R::V + lane * 32);
    }
};
template <class T> struct Tile<T, 8> {
    Raw8<T> p, g;
    uint2 m, v;
    float sm, sv;
    __device__ __forceinline__ void load(const Place<T, 8>& at, int valid) {
        p.load(at.p, valid); g.load(at.g, valid);
        m = load_codes<false>(at.m, valid);
        v = load_codes<false>(at.v, valid);
        sm = *at.sm; sv = *at.sv;
    }
    __device__ __forceinline__ void read(uint32_t stage, int lane) {
        using R = Ring<T, 8>;
        p.read(stage + R::P + lane * 8 * sizeof(T)); g.read(stage + R::G + lane * 8 * sizeof(T));
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(m.x), "=r"(m.y) : "r"(stage + R::M + lane * 8) : "memory");
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(stage + R::V + lane * 8) : "memory");
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(sm), "=f"(sv) : "r"(stage + R::S) : "memory");
    }
};
__device__ __forceinline__ int valid_at(long long n, long long at) { return n - at >= 8 ? 8 : n > at ? (int)(n - at) : 0; }

// The numbers of a step: size = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t), keep = 1 - lr wd.
struct StepNumbers { float size, root, keep, scale; };

template <class T, int BITS, bool FLUSH, bool WHOLE>
__device__ __forceinline__ void update(const Place<T, BITS>& at, const Tile<T, BITS>& tile, int valid, const Hyper& h, const StepNumbers& n) {
    uint64_t p[4], g[4], m[4], v[4];
    tile.p.pairs(p);
    tile.g.pairs(g);
    if constexpr (BITS == 32) {
        tile.m.pairs(m);
        tile.v.pairs(v);
    } else {
        decode<true>(tile.m, tile.sm, m);
        decode<false>(tile.v, tile.sv, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // Sums are scalar here, and each operation rounds by itself: a mul.rn.f32x2 and an add.rn.f32x2 behind it come out as one fused
        // multiply-add, whose sum rounds once, and codes would differ from their definition.
        float m0, m1, v0, v1, a0, a1, d0, d1;
        g[i] = mul2(g[i], twice(n.scale));
        unpack2(mul2(m[i], twice(h.b1)), m0, m1);
        unpack2(mul2(g[i], twice(h.c1)), a0, a1);
        m0 = __fadd_rn(m0, a0);
        m1 = __fadd_rn(m1, a1);
        unpack2(mul2(v[i], twice(h.b2)), v0, v1);
        unpack2(mul2(mul2(g[i], g[i]), twice(h.c2)), a0, a1);
        v0 = __fadd_rn(v0, a0);
        v1 = __fadd_rn(v1, a1);
        m[i] = pack2(m0, m1);
        v[i] = pack2(v0, v1);
        unpack2(fma2(pack2(root_of<FLUSH>(v0), root_of<FLUSH>(v1)), twice(n.root), twice(h.eps)), d0, d1);
        p[i] = fma2(mul2(m[i], pack2(reciprocal_of(d0), reciprocal_of(d1))), twice(-n.size), mul2(p[i], twice(n.keep)));
    }
    store8<WHOLE>(at.p, valid, p);
    if constexpr (BITS == 32) {
        store8<WHOLE>(at.m, valid, m);
        store8<WHOLE>(at.v, valid, v);
    } else {
        store_block<true, WHOLE>(at.m, at.sm, valid, m);
        store_block<false, WHOLE>(at.v, at.sv, valid, v);
    }
}

template <class T, int BITS, bool FLUSH, int CAP>
__global__ void __launch_bounds__(AW_THREADS, 4) adamw_kernel(const __grid_constant__ Table<CAP> table, const __grid_constant__ Hyper h) {
    const int chunk = blockIdx.x;
    int lo = 0, hi = table.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    const Tensor& t = table.t[lo];
    const long long start = (long long)(chunk - table.first[lo]) * table.tiles * AW_TILE, end = min(t.n, start + (long long)table.tiles * AW_TILE);
    using R = Ring<T, BITS>;
    extern __shared__ uint4 smem[];
    const int lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem) + (threadIdx.x >> 5) * R::WARP;
    Place<T, BITS> at(t, start + threadIdx.x * 8);
    Place<T, BITS> warp(t, start + (threadIdx.x & ~31) * 8);      // of the warp's first element
    const int whole = warp.whole() ? (int)((end - start) / AW_TILE) : 0;      // tiles that are copied in words; the same for all threads
#pragma unroll
    for (int i = 0; i < R::STAGES - 1; ++i) {
        if (i < whole) R::fill(ring + i * R::STAGE, warp, i, lane);
        cp_async_commit();
    }
    const int step = t.step[0] + 1;
    // 1 - b^t through expm1, which keeps its digits where b^t is near 1
    const float lr = h.lr_device != nullptr ? *h.lr_device : h.lr;
    const StepNumbers n{lr / -expm1f((float)step * h.ln_b1), rsqrtf(-expm1f((float)step * h.ln_b2)), 1.f - lr * h.wd,
                        h.grad_scale != nullptr ? *h.grad_scale : 1.f};

    Tile<T, BITS> tile;
    for (int i = 0; i < whole; ++i) {
        __syncwarp();      // all lanes have read the stage that is filled now
        if (i + R::STAGES - 1 < whole) R::fill(ring + (i + R::STAGES - 1) % R::STAGES * R::STAGE, warp, R::STAGES - 1, lane);
        cp_async_commit();
        cp_async_wait<R::STAGES - 1>();
        __syncwarp();      // and all have waited for their copies
        tile.read(ring + i % R::STAGES * R::STAGE, lane);
        update<T, BITS, FLUSH, true>(at, tile, 8, h, n);
        at.advance();
        warp.advance();
    }
    for (long long e = start + (long long)whole * AW_TILE + threadIdx.x * 8; (e & ~(long long)(AW_BLOCK - 1)) < end; e += AW_TILE) {      // whole warps
        const int valid = valid_at(t.n, e);
        tile.load(at, valid);
        update<T, BITS, FLUSH, false>(at, tile, valid, h, n);
        at.advance();
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
    constexpr int TILES = 4;
    const long long first = (long long)blockIdx.x * TILES * AW_TILE + threadIdx.x * 8;
    const bool whole = aligned_to(codes, 8) && aligned_to(values, 32);
    uint2 c[TILES];
    float sc[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const long long at = first + i * AW_TILE;
        if (at >= n) continue;
        const int valid = valid_at(n, at);
        c[i] = whole && valid == 8 ? load_codes<true>(codes + at, 8) : load_codes<false>(codes + at, valid);
        sc[i] = scales[at / AW_BLOCK];
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const long long at = first + i * AW_TILE;
        if (at >= n) break;
        const int valid = valid_at(n, at);
        uint64_t x[4];
        decode<SIGNED>(c[i], sc[i], x);
        if (whole && valid == 8) store8<true>(values + at, 8, x);
        else store8<false>(values + at, valid, x);
    }
}

template <class T, int BITS, bool FLUSH, int CAP> int launch_kernel(const Table<CAP>& table, const Hyper& h, unsigned chunks, cudaStream_t s) {
    const auto kernel = adamw_kernel<T, BITS, FLUSH, CAP>;
    const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), Ring<T, BITS>::BYTES);
    if (st != ADDER_OK) return st;
    kernel<<<chunks, AW_THREADS, Ring<T, BITS>::BYTES, s>>>(table, h);
    return launched();
}

// Launches over as many tensors from `tensors` on as a table takes; *next is the first that is left.
template <class T, int CAP> int launch_some(const Tensor* tensors, int count, int* next, const Hyper& h, int bits, bool flush, int tiles, cudaStream_t s) {
    Table<CAP> table;
    table.count = 0;
    table.tiles = tiles;
    const long long elements = (long long)tiles * AW_TILE;
    long long chunks = 0;
    int i = *next;
    for (; i < count && table.count < CAP; ++i) {
        if (tensors[i].n == 0) continue;
        const long long more = (tensors[i].n + elements - 1) / elements;
        if (chunks + more > 2147483647LL) break;
        table.first[table.count] = (int)chunks;
        table.t[table.count++] = tensors[i];
        chunks += more;
    }
    *next = i;
    if (table.count == 0) return ADDER_OK;
    table.first[table.count] = (int)chunks;
    if (bits == 32) return launch_kernel<T, 32, false, CAP>(table, h, (unsigned)chunks, s);
    return flush ? launch_kernel<T, 8, true, CAP>(table, h, (unsigned)chunks, s) : launch_kernel<T, 8, false, CAP>(table, h, (unsigned)chunks, s);
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_adamw_step(const adder_b200_adamw_tensor* tensors, int count, int dtype, int state_bits, double lr, const float* lr_device,
                          double beta1, double beta2, double eps, double weight_decay, const float* grad_scale, void* stream) {
    if (count < 0 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !std::isfinite(lr) ||
        !std::isfinite(weight_decay) || !std::isfinite(eps) || (eps > 0.0 && eps < 0x1p-126))
        return ADDER_ERR_BAD_SHAPE;
    if (state_bits != 32 && state_bits != 8) return ADDER_ERR_UNSUPPORTED;
    if (count == 0) return ADDER_OK;
    if (tensors == nullptr) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(lr_device, 4) || !aligned_to(grad_scale, 4)) return ADDER_ERR_ALIGNMENT;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    long long elements = 0;
    for (int i = 0; i < count; ++i) {
        const adder_b200_adamw_tensor& t = tensors[i];
        if (t.n < 0) return ADDER_ERR_BAD_SHAPE;
        if (t.n == 0) continue;
        if (t.n > 2147483647LL * AW_TILE) return ADDER_ERR_UNSUPPORTED;
        elements += t.n;
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
    // Small models get a CTA for every tile, so that all SMs take part; larger ones up to 4 tiles a CTA, which fetches one while it computes
    // another, and 8 with 8-bit states, which compute longer.  fp32 with 1, 2, 4 and 8 tiles, us: 0.5 M elements 6.3, 6.3, 7.3, 10.2; 1 M 8.7, 8.3,
    // 8.3, 10.4; 3.1 M 17.4, 14.5, 12.4, 14.5; 25 M 119, 110, 109, 112.  bf16 with 8-bit states: 6 M 22.7, 18.6, 17.6, 20.6; 24 M 83, 64, 57, 55.
    int tiles = 1;
    while (tiles < 4 && elements >= 2LL * sm_count() * tiles * AW_TILE) tiles *= 2;
    if (state_bits == 8 && elements >= 32LL * sm_count() * AW_TILE) tiles = 8;
    // Roots of v below 2^-126 are at most 2^-63 / sqrt(1 - beta2^t): where that is below 2^-24 of eps, 8-bit steps take roots that flush (201 M bf16
    // elements 390 us, 411 with the others; 32-bit steps, which memory bounds, take as long either way and have the others alone).
    const bool flush = eps >= 0x1p-39 / std::sqrt(1.0 - beta2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        for (int next = 0; next < count;) {
            const int left = count - next;
            const int st = left <= 48 ? launch_some<T, 48>(tensors, count, &next, h, state_bits, flush, tiles, s)
                           : left <= 176 ? launch_some<T, 176>(tensors, count, &next, h, state_bits, flush, tiles, s)
                                         : launch_some<T, 480>(tensors, count, &next, h, state_bits, flush, tiles, s);
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
    const long long grid = (n + 4 * AW_TILE - 1) / (4 * AW_TILE);
    if (grid > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (is_signed) adamw_values_kernel<true><<<(unsigned)grid, AW_THREADS, 0, s>>>(codes, scales, values, n);
    else adamw_values_kernel<false><<<(unsigned)grid, AW_THREADS, 0, s>>>(codes, scales, values, n);
    return launched();
}

}  // extern "C"
