// Kernels of layer norm and RMS norm over the last axis, forward and backward, with the sum of a residual stream before it.  Each of
// the two includes this file with its NORM_RMS: an RMS norm has no mean and no bias, so what belongs to them is left out.
#pragma once
#include "kernels.h"
#include "e4m3.cuh"
#include "launch.cuh"
#include <cooperative_groups.h>
#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>
#include <initializer_list>
#include <type_traits>

namespace adder {
namespace {

namespace cg = cooperative_groups;

constexpr int NORM_SUMS = NORM_RMS ? 1 : 2;      // sums over the rows: gradients of the weight and the bias

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
    float* scales;             // of codes in y, [rows][blocks]
    long long y_stride;        // of codes in y
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
    } else if constexpr (N == 2 && sizeof(T) == 2) {
        const float2 v = unpack_pair<T>(__ldg(reinterpret_cast<const unsigned*>(p)));
        f[0] = v.x; f[1] = v.y;
    } else if constexpr (N == 2) {
        const float2 v = __ldg(reinterpret_cast<const float2*>(p));
        f[0] = v.x; f[1] = v.y;
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
    else if constexpr (N == 2) *reinterpret_cast<unsigned*>(p) = pack_pair<T>(f[0], f[1]);
    else *reinterpret_cast<uint4*>(p) = Vec16<T>::pack(f);
}

// Sum over the threads of a CTA; `part` is free again after the next barrier.
template <int G> __device__ __forceinline__ float team_sum(float v, float* part, int t) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((t & 31) == 0) part[t >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < G / 32; ++i) v += part[i];
    return v;
}

// Vectors of a row that belong to a CTA of a cluster (all, without one): first and end.
template <bool CLUSTER> __device__ __forceinline__ int2 share_of(int nvec) {
    if constexpr (!CLUSTER) return make_int2(0, nvec);
    const long long rank = cg::this_cluster().block_rank(), parts = cg::this_cluster().num_blocks();
    return make_int2((int)(nvec * rank / parts), (int)(nvec * (rank + 1) / parts));
}

template <int TEAMS, int G> __device__ __forceinline__ void team_barrier(int team) {
    if constexpr (G == 32) __syncwarp();
    else if constexpr (TEAMS == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(G) : "memory");
}

// Shapes of the kernels that hold rows in registers: a team of G threads a row (times the cluster's size), NV vectors of VEC consecutive
// elements a thread.  STAGES > 0: CTAs that stay, a thread's next STAGES - 1 rows on their way through shared memory; a thread copies what it
// reads itself, so only the sums of a row need a barrier.  STAGES = 0: a row a team, and many CTAs an SM (or, with 512 threads, CTAs that
// stay, without the copies).
template <class T_, class W_, int G_, int VEC_, int NV_, int STAGES_, bool CLUSTER_, int THREADS_ = 256> struct LnShape {
    using T = T_;
    using W = W_;
    static constexpr int G = G_, VEC = VEC_, NV = NV_, STAGES = STAGES_;
    static constexpr bool CLUSTER = CLUSTER_;
    static constexpr int THREADS = G > THREADS_ ? G : THREADS_, TEAMS = THREADS / G, WARPS = G / 32;
    static __host__ __device__ constexpr int line() { return THREADS * 16; }      // bytes of one vector of each thread
    static size_t ring(int arrays) { return (size_t)STAGES * arrays * NV * line(); }
};

// A thread's values of a row are held as pairs of fp32, which one instruction adds or multiplies: P pairs of each vector, or, element by
// element, of two elements.
template <class S> struct LnPairs {
    static constexpr int P = S::NV * S::VEC / 2;
    uint64_t p[P];
};
// Whether the pair's vector (element by element: its first element) is in the row.
template <class S> __device__ __forceinline__ bool ln_in(int pair, int v, int v1) { return v + (2 * pair / S::VEC) * S::G < v1; }

// Copies of one array's part of a row into a thread's slots, and out of them; zeros where there is no element.
template <class S> __device__ __forceinline__ void ln_issue(uint32_t slot, const typename S::T* row, int v, int v1) {
#pragma unroll
    for (int i = 0; i < S::NV; ++i)
        if (v + i * S::G < v1)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(slot + i * S::line()), "l"(row + (size_t)(v + i * S::G) * S::VEC) : "memory");
}
template <class S> __device__ __forceinline__ void ln_fetch(LnPairs<S>& f, uint32_t slot, const typename S::T* row, int v, int v1) {
    using T = typename S::T;
    if constexpr (S::STAGES > 0) {
        uint4 q[S::NV];
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            q[i] = make_uint4(0, 0, 0, 0);
            if (v + i * S::G < v1)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[i].x), "=r"(q[i].y), "=r"(q[i].z), "=r"(q[i].w) : "r"(slot + i * S::line()) : "memory");
        }
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            float e[S::VEC];
            Vec16<T>::unpack(q[i], e);
#pragma unroll
            for (int j = 0; j < S::VEC; j += 2) f.p[(i * S::VEC + j) / 2] = pack2(e[j], e[j + 1]);
        }
    } else {
        float e[S::NV][S::VEC];
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
#pragma unroll
            for (int j = 0; j < S::VEC; ++j) e[i][j] = 0.f;
            if (v + i * S::G < v1) load_some<T, S::VEC>(row + (size_t)(v + i * S::G) * S::VEC, e[i]);
        }
#pragma unroll
        for (int i = 0; i < LnPairs<S>::P; ++i) f.p[i] = pack2((&e[0][0])[2 * i], (&e[0][0])[2 * i + 1]);
    }
}
template <class S> __device__ __forceinline__ void ln_store(typename S::T* row, const LnPairs<S>& f, int v, int v1) {
    float e[S::NV][S::VEC];
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) unpack2(f.p[i], (&e[0][0])[2 * i], (&e[0][0])[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < S::NV; ++i)
        if (v + i * S::G < v1) store_some<typename S::T, S::VEC>(row + (size_t)(v + i * S::G) * S::VEC, e[i]);
}
template <class S> __device__ __forceinline__ void ln_weights(LnPairs<S>& f, const void* w, float missing, int v, int v1) {
    float e[S::NV][S::VEC];
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
#pragma unroll
        for (int j = 0; j < S::VEC; ++j) e[i][j] = missing;
        if (w != nullptr && v + i * S::G < v1) load_some<typename S::W, S::VEC>(static_cast<const typename S::W*>(w) + (size_t)(v + i * S::G) * S::VEC, e[i]);
    }
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) f.p[i] = pack2((&e[0][0])[2 * i], (&e[0][0])[2 * i + 1]);
}

// Which rows a team takes, and the ring of the rows on their way.
template <class S> struct LnWalk {
    long long row, ahead, step;      // the next to be read, the next to be copied
    uint32_t ring, fill, read;       // bytes
    int arrays;

    __device__ __forceinline__ void start(void* smem, int arrays_) {
        row = ahead = (long long)blockIdx.x * S::TEAMS + threadIdx.x / S::G;
        step = (long long)gridDim.x * S::TEAMS;
        ring = fill = read = smem_u32(smem) + threadIdx.x * 16;
        arrays = arrays_;
    }
    __device__ __forceinline__ uint32_t advance(uint32_t at) const {
        const uint32_t stage = (uint32_t)arrays * S::NV * S::line(), last = S::STAGES > 0 ? S::STAGES - 1 : 0;
        return at == ring + last * stage ? ring : at + stage;
    }
    static __device__ __forceinline__ uint32_t slot(uint32_t at, int array) { return at + array * S::NV * S::line(); }
};

// Exchange of a row's sums between the warps of a team, and between the CTAs of a cluster.
template <class S> struct LnSums {
    float2 part[2][S::TEAMS][S::WARPS];
    float2 ranks[2][8];
    float2 count[S::WARPS];      // elements of a row that each warp holds, and one over that (0 where it holds none)
    float2 rank_count[8];        // and each CTA of the cluster
};

__device__ __forceinline__ float2 count_of(int n) { return make_float2((float)n, n > 0 ? 1.f / (float)n : 0.f); }
template <class S> __device__ __forceinline__ void ln_count(LnSums<S>& sh, int v0, int v1, int nvec) {
    if constexpr (NORM_RMS) return;      // no means to be joined
    if (threadIdx.x < S::WARPS) {
        int n = 0;
        for (int i = 0; i < S::NV; ++i) n += max(0, min(32, v1 - (v0 + i * S::G + 32 * (int)threadIdx.x)));
        sh.count[threadIdx.x] = count_of(n * S::VEC);
    }
    if constexpr (S::CLUSTER) {
        const long long parts = cg::this_cluster().num_blocks(), i = threadIdx.x;
        if (i < parts) sh.rank_count[i] = count_of((int)(nvec * (i + 1) / parts - nvec * i / parts) * S::VEC);
    }
    __syncthreads();
}
// The CTAs of a cluster tell one another that they have begun, and wait for that before the first word crosses over.
template <bool CLUSTER> __device__ __forceinline__ void cluster_arrive() {
    if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
}
template <bool CLUSTER> __device__ __forceinline__ void cluster_wait() {
    if constexpr (CLUSTER) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
// A pair (a, b) of every warp of the team, in lane i % WARPS of every warp that of warp i.  `turn` alternates, so that one barrier a row is
// enough: who writes a row's pairs has seen the barrier after all had read those of the row before the last.
template <class S> __device__ __forceinline__ float2 ln_exchange(float a, float b, LnSums<S>& sh, int team, int t, int turn) {
    if ((t & 31) == 0) sh.part[turn][team][t >> 5] = make_float2(a, b);
    team_barrier<S::TEAMS, S::G>(team);
    return sh.part[turn][team][t % S::WARPS];
}
// The same over the CTAs of a cluster, in lane i % 8; zeros beyond its size.  Once in a kernel: what is written to a CTA is there when it
// passes the barrier, after which it may leave.
template <class S> __device__ __forceinline__ float2 ln_exchange_ranks(float a, float b, LnSums<S>& sh, int t, int turn) {
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks();
    if (t < parts) cluster.map_shared_rank(&sh.ranks[turn][0], t)[cluster.block_rank()] = make_float2(a, b);
    cluster.sync();
    return t % 8 < parts ? sh.ranks[turn][t % 8] : make_float2(0.f, 0.f);
}

// Two sums at once, over all threads that share the row.
template <class S> __device__ __forceinline__ float2 ln_sum2(float a, float b, LnSums<S>& sh, int team, int t, int turn) {
    a = lanes_sum<32>(a);
    b = lanes_sum<32>(b);
    if constexpr (S::WARPS > 1) {
        const float2 p = ln_exchange<S>(a, b, sh, team, t, turn);
        a = lanes_sum<S::WARPS>(p.x);
        b = lanes_sum<S::WARPS>(p.y);
    }
    if constexpr (S::CLUSTER) {
        const float2 p = ln_exchange_ranks<S>(a, b, sh, t, turn);
        a = lanes_sum<8>(p.x);
        b = lanes_sum<8>(p.y);
    }
    return make_float2(a, b);
}

// One sum over all threads that share the row.
template <class S> __device__ __forceinline__ float ln_sum1(float a, LnSums<S>& sh, int team, int t, int turn) {
    a = lanes_sum<32>(a);
    if constexpr (S::WARPS > 1) a = lanes_sum<S::WARPS>(ln_exchange<S>(a, 0.f, sh, team, t, turn).x);
    if constexpr (S::CLUSTER) a = lanes_sum<8>(ln_exchange_ranks<S>(a, 0.f, sh, t, turn).x);
    return a;
}

// Mean and sum of squared differences from it: each warp has both of its own elements, and what the warps' means differ from the whole one
// by comes on top, so one barrier does and nothing cancels.
template <class S> __device__ __forceinline__ float2 ln_moments(const LnPairs<S>& f, int v, int v1, float inv_d, LnSums<S>& sh, int team, int t, int turn) {
    if constexpr (NORM_RMS) {      // squares as they are; zeros where there is no element
        uint64_t sq2 = 0;
#pragma unroll
        for (int i = 0; i < LnPairs<S>::P; ++i) sq2 = fma2(f.p[i], f.p[i], sq2);
        float lo, hi;
        unpack2(sq2, lo, hi);
        return make_float2(0.f, ln_sum1<S>(lo + hi, sh, team, t, turn));
    }
    uint64_t sum2 = 0;
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) sum2 = add2(sum2, f.p[i]);      // zeros where there is no element
    float lo, hi;
    unpack2(sum2, lo, hi);
    const float sum = lanes_sum<32>(lo + hi);
    constexpr bool one = S::WARPS == 1 && !S::CLUSTER;
    const float mine = sum * (one ? inv_d : sh.count[t >> 5].y);
    const uint64_t minus = pack2(-mine, -mine);
    uint64_t sq2 = 0;
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) {
        if constexpr (S::VEC > 1) {
            if (ln_in<S>(i, v, v1)) {
                const uint64_t e = add2(f.p[i], minus);
                sq2 = fma2(e, e, sq2);
            }
        } else {
            float a, b;
            unpack2(add2(f.p[i], minus), a, b);
            const uint64_t e = pack2(v + 2 * i * S::G < v1 ? a : 0.f, v + (2 * i + 1) * S::G < v1 ? b : 0.f);
            sq2 = fma2(e, e, sq2);
        }
    }
    unpack2(sq2, lo, hi);
    float sq = lanes_sum<32>(lo + hi), mean = mine;
    if constexpr (!one) {
        float2 p = ln_exchange<S>(sum, sq, sh, team, t, turn), n = sh.count[t % S::WARPS];
        float all = lanes_sum<S::WARPS>(p.x), held = 0.f;
        if constexpr (S::CLUSTER) held = sh.rank_count[cg::this_cluster().block_rank()].y;
        mean = all * (S::CLUSTER ? held : inv_d);
        float e = p.x * n.y - mean;
        sq = lanes_sum<S::WARPS>(fmaf(n.x * e, e, p.y));
        if constexpr (S::CLUSTER) {
            p = ln_exchange_ranks<S>(all, sq, sh, t, turn);
            n = t % 8 < (int)cg::this_cluster().num_blocks() ? sh.rank_count[t % 8] : make_float2(0.f, 0.f);
            mean = lanes_sum<8>(p.x) * inv_d;
            e = p.x * n.y - mean;
            sq = lanes_sum<8>(fmaf(n.x * e, e, p.y));
        }
    }
    return make_float2(mean, sq);
}

// 1 / sqrt(x), the approximate one and a step of Newton's method; 0 for a variance beyond the range and infinity for 0, which the step
// would turn into NaN.
__device__ __forceinline__ float inverse_root(float x) {
    const float r = rsqrtf(x);
    return r > 0.f && r < INFINITY ? r * fmaf(-0.5f * (x * r), r, 1.5f) : r;
}

__device__ __forceinline__ void ln_keep(const LnFwd& a, long long row, float mean, float rs) {
    if constexpr (!NORM_RMS) a.mean[row] = mean;
    a.rstd[row] = rs;
}

// y in 8 bits: a block of 128 columns lies with 128 / VEC neighbouring lanes, in one vector of each.
template <class S> __device__ __forceinline__ void ln_store_codes(const LnFwd& a, long long row, const LnPairs<S>& f, int v, int v1) {
    constexpr int LANES = E4M3_BLOCK / S::VEC;
    const int blocks = (a.d + E4M3_BLOCK - 1) / E4M3_BLOCK;
    uint8_t* out = static_cast<uint8_t*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
        float e[S::VEC], largest = 0.f;
#pragma unroll
        for (int j = 0; j < S::VEC; j += 2) unpack2(f.p[(i * S::VEC + j) / 2], e[j], e[j + 1]);
#pragma unroll
        for (int j = 0; j < S::VEC; ++j) largest = max_nan(largest, fabsf(e[j]));
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, off));
        const E4m3Scale s = e4m3_scale(largest);
        const int at = v + i * S::G;
        if (at < v1) {
            if constexpr (S::VEC == 8) *reinterpret_cast<uint2*>(out + at * 8) = make_uint2(e4m3_word(e[0], e[1], e[2], e[3], s.inverse), e4m3_word(e[4], e[5], e[6], e[7], s.inverse));
            else *reinterpret_cast<uint32_t*>(out + at * 4) = e4m3_word(e[0], e[1], e[2], e[3], s.inverse);
            if (at % LANES == 0) a.scales[row * blocks + at / LANES] = s.scale;
        }
    }
}

// h = x + residual, rounded to what is stored: the norm is taken of that.
template <class S> __device__ __forceinline__ void ln_add(LnPairs<S>& f, const LnPairs<S>& r) {
    using T = typename S::T;
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) {
        f.p[i] = add2(f.p[i], r.p[i]);
        if constexpr (sizeof(T) == 2) {
            float lo, hi;
            unpack2(f.p[i], lo, hi);
            const float2 held = unpack_pair<T>(pack_pair<T>(lo, hi));
            f.p[i] = pack2(held.x, held.y);
        }
    }
}

template <class S, bool EIGHT> __global__ void __launch_bounds__(S::THREADS, S::THREADS > 256 ? 1 : 3) ln_forward_kernel(const LnFwd a) {
    extern __shared__ uint4 smem[];
    __shared__ LnSums<S> sh;
    using T = typename S::T;
    const int t = threadIdx.x % S::G, team = threadIdx.x / S::G;
    const int v = t, v1 = a.d / S::VEC;
    const float inv_d = 1.f / a.d;
    LnWalk<S> walk;
    walk.start(smem, a.residual != nullptr ? 2 : 1);
    const auto issue = [&] {
        if (walk.ahead < a.rows) {
            ln_issue<S>(walk.slot(walk.fill, 0), static_cast<const T*>(a.x) + walk.ahead * a.x_stride, v, v1);
            if (a.residual != nullptr) ln_issue<S>(walk.slot(walk.fill, 1), static_cast<const T*>(a.residual) + walk.ahead * a.r_stride, v, v1);
            walk.ahead += walk.step;
        }
        cp_async_commit();
        walk.fill = walk.advance(walk.fill);
    };
    for (int i = 0; i < S::STAGES - 1; ++i) issue();
    ln_count<S>(sh, 0, v1, v1);
    LnPairs<S> w, b;
    ln_weights<S>(w, a.w, 1.f, v, v1);
    if constexpr (!NORM_RMS) ln_weights<S>(b, a.b, 0.f, v, v1);
    int turn = 0;
    for (; walk.row < a.rows; walk.row += walk.step) {
        issue();
        cp_async_wait<S::STAGES - 1>();
        const long long row = walk.row;
        LnPairs<S> f;
        ln_fetch<S>(f, walk.slot(walk.read, 0), nullptr, v, v1);
        if (a.residual != nullptr) {
            LnPairs<S> r;
            ln_fetch<S>(r, walk.slot(walk.read, 1), nullptr, v, v1);
            ln_add<S>(f, r);
            ln_store<S>(static_cast<T*>(a.h) + row * a.d, f, v, v1);
        }
        walk.read = walk.advance(walk.read);
        const float2 mom = ln_moments<S>(f, v, v1, inv_d, sh, team, t, turn);
        turn ^= 1;
        const float rs = inverse_root(mom.y * inv_d + a.eps);
        if (a.rstd != nullptr && t == 0) ln_keep(a, row, mom.x, rs);
        const uint64_t minus = pack2(-mom.x, -mom.x), scale = pack2(rs, rs);
#pragma unroll
        for (int i = 0; i < LnPairs<S>::P; ++i) {
            if constexpr (NORM_RMS) f.p[i] = mul2(mul2(f.p[i], scale), w.p[i]);
            else f.p[i] = fma2(mul2(add2(f.p[i], minus), scale), w.p[i], b.p[i]);
        }
        if constexpr (EIGHT) ln_store_codes<S>(a, row, f, v, v1);
        else ln_store<S>(static_cast<T*>(a.y) + row * a.d, f, v, v1);
    }
}

template <class S> __global__ void __launch_bounds__(S::THREADS, S::NV * S::VEC <= 16 ? 4 : S::VEC > 2 ? 3 : 2) ln_forward_row_kernel(const LnFwd a) {
    __shared__ LnSums<S> sh;
    cluster_arrive<S::CLUSTER>();
    using T = typename S::T;
    const int t = threadIdx.x % S::G, team = threadIdx.x / S::G;
    const int2 share = share_of<S::CLUSTER>(a.d / S::VEC);
    const int v = share.x + t, v1 = share.y;
    const float inv_d = 1.f / a.d;
    const long long parts = S::CLUSTER ? (long long)cg::this_cluster().num_blocks() : 1;
    const long long row = blockIdx.x / parts * S::TEAMS + team;
    LnPairs<S> f;
    if (row < a.rows) {
        ln_fetch<S>(f, 0, static_cast<const T*>(a.x) + row * a.x_stride, v, v1);
        if (a.residual != nullptr) {
            LnPairs<S> r;
            ln_fetch<S>(r, 0, static_cast<const T*>(a.residual) + row * a.r_stride, v, v1);
            ln_add<S>(f, r);
            ln_store<S>(static_cast<T*>(a.h) + row * a.d, f, v, v1);
        }
    }
    ln_count<S>(sh, share.x, share.y, a.d / S::VEC);
    cluster_wait<S::CLUSTER>();
    if (row < a.rows) {      // the same for all of a team, and for a cluster
        const float2 mom = ln_moments<S>(f, v, v1, inv_d, sh, team, t, 0);
        const float rs = inverse_root(mom.y * inv_d + a.eps);
        if (a.rstd != nullptr && t == 0 && share.x == 0) ln_keep(a, row, mom.x, rs);
        const uint64_t minus = pack2(-mom.x, -mom.x), scale = pack2(rs, rs);
        LnPairs<S> w;
        ln_weights<S>(w, a.w, 1.f, v, v1);
#pragma unroll
        for (int i = 0; i < LnPairs<S>::P; ++i) f.p[i] = mul2(mul2(NORM_RMS ? f.p[i] : add2(f.p[i], minus), scale), w.p[i]);
        if constexpr (!NORM_RMS) {
            ln_weights<S>(w, a.b, 0.f, v, v1);
#pragma unroll
            for (int i = 0; i < LnPairs<S>::P; ++i) f.p[i] = add2(f.p[i], w.p[i]);
        }
        ln_store<S>(static_cast<T*>(a.y) + row * a.d, f, v, v1);
    }
}

// The sums of g and of g xh (of the latter alone without a mean) over the row.
template <class S> __device__ __forceinline__ float2 ln_dots(uint64_t s1, uint64_t s2, LnSums<S>& sh, int team, int t, int turn) {
    float a1, b1, a2, b2;
    unpack2(s1, a1, b1);
    unpack2(s2, a2, b2);
    if constexpr (NORM_RMS) return make_float2(0.f, ln_sum1<S>(a2 + b2, sh, team, t, turn));
    else return ln_sum2<S>(a1 + b1, a2 + b2, sh, team, t, turn);
}
__device__ __forceinline__ float ln_mean(const LnBwd& a, long long row) { return NORM_RMS ? 0.f : a.mean[row]; }

// dx of rows that a cluster shares, a row each.
template <class S> __global__ void __launch_bounds__(S::THREADS, S::NV * S::VEC > 16 ? 2 : 3) ln_dx_row_kernel(const LnBwd a) {
    static_assert(S::CLUSTER && S::TEAMS == 1, "shorter rows go by CTAs that stay");
    __shared__ LnSums<S> sh;
    cluster_arrive<true>();
    using T = typename S::T;
    const int t = threadIdx.x;
    const int2 share = share_of<true>(a.d / S::VEC);
    const int v = share.x + t, v1 = share.y;
    const float inv_d = 1.f / a.d;
    const long long row = blockIdx.x / cg::this_cluster().num_blocks();
    LnPairs<S> xh, g, w;
    const float mean = ln_mean(a, row), rs = a.rstd[row];
    ln_fetch<S>(xh, 0, static_cast<const T*>(a.h) + row * a.h_stride, v, v1);
    ln_fetch<S>(g, 0, static_cast<const T*>(a.dy) + row * a.d, v, v1);
    cluster_wait<true>();
    ln_weights<S>(w, a.w, 1.f, v, v1);
    uint64_t s1 = 0, s2 = 0;
    const uint64_t minus = pack2(-mean, -mean), scale = pack2(rs, rs);
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) {      // dy is 0 where there is no element
        xh.p[i] = mul2(NORM_RMS ? xh.p[i] : add2(xh.p[i], minus), scale);
        g.p[i] = mul2(g.p[i], w.p[i]);
        if constexpr (!NORM_RMS) s1 = add2(s1, g.p[i]);
        s2 = fma2(g.p[i], xh.p[i], s2);
    }
    const float2 m = ln_dots<S>(s1, s2, sh, 0, t, 0);
    const float c1 = -m.x * inv_d, c2 = -m.y * inv_d;
    const uint64_t shift = pack2(c1, c1), slope = pack2(c2, c2);
#pragma unroll
    for (int i = 0; i < LnPairs<S>::P; ++i) g.p[i] = mul2(fma2(xh.p[i], slope, NORM_RMS ? g.p[i] : add2(g.p[i], shift)), scale);
    if (a.dh != nullptr) {
        ln_fetch<S>(w, 0, static_cast<const T*>(a.dh) + row * a.d, v, v1);
#pragma unroll
        for (int i = 0; i < LnPairs<S>::P; ++i) g.p[i] = add2(g.p[i], w.p[i]);
    }
    ln_store<S>(static_cast<T*>(a.dx) + row * a.d, g, v, v1);
}

// dx of every row; with SUMS this thread's columns of dw and db, added up over its rows and then over the CTA's teams into
// part[CTA or cluster][NORM_SUMS][d].
template <class S, bool SUMS> __global__ void __launch_bounds__(S::THREADS, 1) ln_backward_kernel(const LnBwd a, float* part) {
    extern __shared__ uint4 smem[];
    __shared__ LnSums<S> sh;
    using T = typename S::T;
    const int t = threadIdx.x % S::G, team = threadIdx.x / S::G;
    const int v = t, v1 = a.d / S::VEC;
    LnWalk<S> walk;
    walk.start(smem, a.dh != nullptr ? 3 : 2);
    const auto issue = [&] {
        if (walk.ahead < a.rows) {
            ln_issue<S>(walk.slot(walk.fill, 0), static_cast<const T*>(a.h) + walk.ahead * a.h_stride, v, v1);
            ln_issue<S>(walk.slot(walk.fill, 1), static_cast<const T*>(a.dy) + walk.ahead * a.d, v, v1);
            if (a.dh != nullptr) ln_issue<S>(walk.slot(walk.fill, 2), static_cast<const T*>(a.dh) + walk.ahead * a.d, v, v1);
            walk.ahead += walk.step;
        }
        cp_async_commit();
        walk.fill = walk.advance(walk.fill);
    };
    if constexpr (S::STAGES > 0)
        for (int i = 0; i < S::STAGES - 1; ++i) issue();
    constexpr int P = LnPairs<S>::P;
    const float inv_d = 1.f / a.d;
    LnPairs<S> w, dw, db;
    ln_weights<S>(w, a.w, 1.f, v, v1);
#pragma unroll
    for (int i = 0; i < P; ++i) dw.p[i] = db.p[i] = 0;
    float mean = 0.f, rs = 0.f;
    if (walk.row < a.rows) { mean = ln_mean(a, walk.row); rs = a.rstd[walk.row]; }
    int turn = 0;
    for (; walk.row < a.rows; walk.row += walk.step) {
        if constexpr (S::STAGES > 0) {
            issue();
            cp_async_wait<(S::STAGES > 0 ? S::STAGES - 1 : 0)>();
        }
        const long long row = walk.row, next = row + walk.step;
        float mean_next = 0.f, rs_next = 0.f;
        if (next < a.rows) { mean_next = ln_mean(a, next); rs_next = a.rstd[next]; }
        LnPairs<S> xh, g;
        ln_fetch<S>(xh, walk.slot(walk.read, 0), static_cast<const T*>(a.h) + row * a.h_stride, v, v1);
        ln_fetch<S>(g, walk.slot(walk.read, 1), static_cast<const T*>(a.dy) + row * a.d, v, v1);
        uint64_t s1 = 0, s2 = 0;
        const uint64_t minus = pack2(-mean, -mean), scale = pack2(rs, rs);
#pragma unroll
        for (int i = 0; i < P; ++i) {      // dy is 0 where there is no element
            xh.p[i] = mul2(NORM_RMS ? xh.p[i] : add2(xh.p[i], minus), scale);
            if (SUMS) {
                dw.p[i] = fma2(g.p[i], xh.p[i], dw.p[i]);
                if constexpr (!NORM_RMS) db.p[i] = add2(db.p[i], g.p[i]);
            }
            g.p[i] = mul2(g.p[i], w.p[i]);
            if constexpr (!NORM_RMS) s1 = add2(s1, g.p[i]);
            s2 = fma2(g.p[i], xh.p[i], s2);
        }
        if (a.dx != nullptr) {
            const float2 m = ln_dots<S>(s1, s2, sh, team, t, turn);
            turn ^= 1;
            const float c1 = -m.x * inv_d, c2 = -m.y * inv_d;
            const uint64_t shift = pack2(c1, c1), slope = pack2(c2, c2);
#pragma unroll
            for (int i = 0; i < P; ++i) g.p[i] = mul2(fma2(xh.p[i], slope, NORM_RMS ? g.p[i] : add2(g.p[i], shift)), scale);
            if (a.dh != nullptr) {
                LnPairs<S> e;
                ln_fetch<S>(e, walk.slot(walk.read, 2), static_cast<const T*>(a.dh) + row * a.d, v, v1);
#pragma unroll
                for (int i = 0; i < P; ++i) g.p[i] = add2(g.p[i], e.p[i]);
            }
            ln_store<S>(static_cast<T*>(a.dx) + row * a.d, g, v, v1);
        }
        if constexpr (S::STAGES > 0) walk.read = walk.advance(walk.read);
        mean = mean_next; rs = rs_next;
    }
    if constexpr (SUMS) {
        float* out = part + (size_t)blockIdx.x * NORM_SUMS * a.d;
        // one team writes its sums to the workspace, several add them up in their order, in shared memory
        float* to = out;
        if constexpr (S::TEAMS > 1) {
            cp_async_wait<0>();
            __syncthreads();
            to = reinterpret_cast<float*>(smem) + team * NORM_SUMS * a.d;
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float lo, hi;
            const int c = S::VEC > 1 ? (v + 2 * i / S::VEC * S::G) * S::VEC + 2 * i % S::VEC : v + 2 * i * S::G, c2 = S::VEC > 1 ? c + 1 : c + S::G;
            const bool in = ln_in<S>(i, v, v1), in2 = S::VEC > 1 ? in : c2 < v1;
            unpack2(dw.p[i], lo, hi);
            if (in) to[c] = lo;
            if (in2) to[c2] = hi;
            if constexpr (!NORM_RMS) {
                unpack2(db.p[i], lo, hi);
                if (in) to[a.d + c] = lo;
                if (in2) to[a.d + c2] = hi;
            }
        }
        if constexpr (S::TEAMS > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < NORM_SUMS * a.d; c += S::THREADS) {
                float sum = 0.f;
                for (int i = 0; i < S::TEAMS; ++i) sum += reinterpret_cast<float*>(smem)[i * NORM_SUMS * a.d + c];
                out[c] = sum;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ long rows, held in shared memory

// One CTA an SM, which has a row and the next one in shared memory: with enough rows for all SMs nothing is exchanged between CTAs.  A
// thread copies the vectors that it reads itself.
constexpr int LN_WIDE = 1024;

template <class T> __device__ __forceinline__ void wide_copy(uint4* to, const T* row, int nvec) {
    const uint32_t base = smem_u32(to);
    for (int v = threadIdx.x; v < nvec; v += LN_WIDE)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(base + 16 * v), "l"(row + (size_t)v * Vec16<T>::N) : "memory");
}
// Sums over the CTA; `part` alternates between two arrays.
__device__ __forceinline__ float2 wide_sum2(float a, float b, float2* part) {
    a = lanes_sum<32>(a);
    b = lanes_sum<32>(b);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 p = part[threadIdx.x & 31];
    return make_float2(lanes_sum<32>(p.x), lanes_sum<32>(p.y));
}
template <class T> __device__ __forceinline__ void vector_pairs(const uint4& q, uint64_t (&f)[Vec16<T>::N / 2]) {
    float e[Vec16<T>::N];
    Vec16<T>::unpack(q, e);
#pragma unroll
    for (int i = 0; i < Vec16<T>::N / 2; ++i) f[i] = pack2(e[2 * i], e[2 * i + 1]);
}
template <class T> __device__ __forceinline__ uint4 pairs_vector(const uint64_t (&f)[Vec16<T>::N / 2]) {
    float e[Vec16<T>::N];
#pragma unroll
    for (int i = 0; i < Vec16<T>::N / 2; ++i) unpack2(f[i], e[2 * i], e[2 * i + 1]);
    return Vec16<T>::pack(e);
}
template <class W, int N> __device__ __forceinline__ void weight_pairs(const void* w, float missing, int v, uint64_t (&f)[N / 2]) {
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = missing;
    if (w != nullptr) load_some<W, N>(static_cast<const W*>(w) + (size_t)v * N, e);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i] = pack2(e[2 * i], e[2 * i + 1]);
}

template <class T, class W> __global__ void __launch_bounds__(LN_WIDE) ln_forward_wide_kernel(const LnFwd a) {
    extern __shared__ uint4 smem[];
    __shared__ float2 part[2][LN_WIDE / 32];
    constexpr int N = Vec16<T>::N, P = N / 2;
    const int nvec = a.d / N, arrays = a.residual != nullptr ? 2 : 1;
    const float inv_d = 1.f / a.d;
    const auto issue = [&](long long row, uint4* to) {
        if (row < a.rows) {
            wide_copy<T>(to, static_cast<const T*>(a.x) + row * a.x_stride, nvec);
            if (arrays == 2) wide_copy<T>(to + nvec, static_cast<const T*>(a.residual) + row * a.r_stride, nvec);
        }
        cp_async_commit();
    };
    long long row = blockIdx.x;
    issue(row, smem);
    for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
        uint4* held = smem + turn * arrays * nvec;
        issue(row + gridDim.x, smem + (turn ^ 1) * arrays * nvec);
        cp_async_wait<1>();
        uint64_t sum = 0;
        for (int v = threadIdx.x; v < nvec; v += LN_WIDE) {
            uint64_t f[P];
            vector_pairs<T>(held[v], f);
            if (arrays == 2) {
                uint64_t r[P];
                vector_pairs<T>(held[nvec + v], r);
#pragma unroll
                for (int i = 0; i < P; ++i) f[i] = add2(f[i], r[i]);
                const uint4 h = pairs_vector<T>(f);      // rounded: the norm is taken of what is stored
                held[v] = h;
                reinterpret_cast<uint4*>(static_cast<T*>(a.h) + row * a.d)[v] = h;
                vector_pairs<T>(h, f);
            }
#pragma unroll
            for (int i = 0; i < P; ++i) sum = NORM_RMS ? fma2(f[i], f[i], sum) : add2(sum, f[i]);
        }
        float lo, hi;
        unpack2(sum, lo, hi);
        const float first = wide_sum2(lo + hi, 0.f, part[NORM_RMS ? turn : 0]).x, mean = NORM_RMS ? 0.f : first * inv_d;
        const uint64_t minus = pack2(-mean, -mean);
        float squares = first;
        if constexpr (!NORM_RMS) {
            uint64_t sq = 0;
            for (int v = threadIdx.x; v < nvec; v += LN_WIDE) {
                uint64_t f[P];
                vector_pairs<T>(held[v], f);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const uint64_t e = add2(f[i], minus);
                    sq = fma2(e, e, sq);
                }
            }
            unpack2(sq, lo, hi);
            squares = wide_sum2(lo + hi, 0.f, part[1]).x;
        }
        const float rs = inverse_root(squares * inv_d + a.eps);
        if (a.rstd != nullptr && threadIdx.x == 0) ln_keep(a, row, mean, rs);
        const uint64_t scale = pack2(rs, rs);
#pragma unroll 2
        for (int v = threadIdx.x; v < nvec; v += LN_WIDE) {
            uint64_t f[P], w[P], b[P];
            weight_pairs<W, N>(a.w, 1.f, v, w);
            if constexpr (!NORM_RMS) weight_pairs<W, N>(a.b, 0.f, v, b);
            vector_pairs<T>(held[v], f);
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = NORM_RMS ? mul2(mul2(f[i], scale), w[i]) : fma2(mul2(add2(f[i], minus), scale), w[i], b[i]);
            reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.d)[v] = pairs_vector<T>(f);
        }
    }
}

template <class T, class W> __global__ void __launch_bounds__(LN_WIDE) ln_dx_wide_kernel(const LnBwd a) {
    extern __shared__ uint4 smem[];
    __shared__ float2 part[2][LN_WIDE / 32];
    constexpr int N = Vec16<T>::N, P = N / 2;
    const int nvec = a.d / N;
    const float inv_d = 1.f / a.d;
    const auto issue = [&](long long row, uint4* to) {
        if (row < a.rows) {
            wide_copy<T>(to, static_cast<const T*>(a.h) + row * a.h_stride, nvec);
            wide_copy<T>(to + nvec, static_cast<const T*>(a.dy) + row * a.d, nvec);
        }
        cp_async_commit();
    };
    long long row = blockIdx.x;
    issue(row, smem);
    for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
        const uint4* held = smem + turn * 2 * nvec;
        const float mean = ln_mean(a, row), rs = a.rstd[row];
        issue(row + gridDim.x, smem + (turn ^ 1) * 2 * nvec);
        cp_async_wait<1>();
        const uint64_t minus = pack2(-mean, -mean), scale = pack2(rs, rs);
        uint64_t s1 = 0, s2 = 0;
        const auto both = [&](int v, uint64_t (&xh)[P], uint64_t (&g)[P]) {
            uint64_t w[P];
            weight_pairs<W, N>(a.w, 1.f, v, w);
            vector_pairs<T>(held[v], xh);
            vector_pairs<T>(held[nvec + v], g);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                xh[i] = mul2(NORM_RMS ? xh[i] : add2(xh[i], minus), scale);
                g[i] = mul2(g[i], w[i]);
            }
        };
#pragma unroll 2
        for (int v = threadIdx.x; v < nvec; v += LN_WIDE) {
            uint64_t xh[P], g[P];
            both(v, xh, g);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if constexpr (!NORM_RMS) s1 = add2(s1, g[i]);
                s2 = fma2(g[i], xh[i], s2);
            }
        }
        float a1, b1, a2, b2;
        unpack2(s1, a1, b1);
        unpack2(s2, a2, b2);
        const float2 m = wide_sum2(a1 + b1, a2 + b2, part[turn]);
        const float c1 = -m.x * inv_d, c2 = -m.y * inv_d;
        const uint64_t shift = pack2(c1, c1), slope = pack2(c2, c2);
#pragma unroll 2
        for (int v = threadIdx.x; v < nvec; v += LN_WIDE) {
            uint64_t xh[P], g[P];
            both(v, xh, g);
#pragma unroll
            for (int i = 0; i < P; ++i) g[i] = mul2(fma2(xh[i], slope, NORM_RMS ? g[i] : add2(g[i], shift)), scale);
            if (a.dh != nullptr) {
                uint64_t e[P];
                weight_pairs<T, N>(static_cast<const T*>(a.dh) + row * a.d, 0.f, v, e);
#pragma unroll
                for (int i = 0; i < P; ++i) g[i] = add2(g[i], e[i]);
            }
            reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.d)[v] = pairs_vector<T>(g);
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
    float sq = 0.f, mean = 0.f;
    if constexpr (!NORM_RMS) {
        float sum = 0.f;
        for (int c = c0 + t; c < c1; c += LN_LONG) sum += at(c);
        mean = cluster_sum(sum, part[0], slot, t) / a.d;
    }
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float e = at(c) - mean;
        sq += e * e;
    }
    const float rs = 1.f / sqrtf(cluster_sum(sq, part[1], slot + 1, t) / a.d + a.eps);
    if (t == 0 && rank == 0 && a.rstd != nullptr) ln_keep(a, row, mean, rs);
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
    const float mean = ln_mean(a, row), rs = a.rstd[row];
    const int c0 = (int)((long long)a.d * rank / parts), c1 = (int)((long long)a.d * (rank + 1) / parts);
    const auto weight = [&](int c) { return a.w != nullptr ? to_float(static_cast<const W*>(a.w)[c]) : 1.f; };
    float s1 = 0.f, s2 = 0.f;
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float g = to_float(dy[c]) * weight(c);
        s1 += g;
        s2 = fmaf(g, (to_float(h[c]) - mean) * rs, s2);
    }
    s1 = NORM_RMS ? 0.f : cluster_sum(s1, part[0], slot, t) / a.d;
    s2 = cluster_sum(s2, part[1], slot + 1, t) / a.d;
    for (int c = c0 + t; c < c1; c += LN_LONG) {
        const float o = rs * (to_float(dy[c]) * weight(c) - s1 - (to_float(h[c]) - mean) * rs * s2);
        dx[c] = from_float<T>(dh != nullptr ? o + to_float(dh[c]) : o);
    }
    cg::this_cluster().sync();
}

// ------------------------------------------------------------------------------------------ gradients of weight and bias

constexpr int LN_COLS = 32, LN_LINES = 8;      // a CTA's columns (of VEC elements), and the rows that it reads at once

// grid (column tiles, splits): part[split][NORM_SUMS][d]
template <class T, int VEC> __global__ void __launch_bounds__(LN_COLS * LN_LINES) ln_columns_kernel(const LnBwd a, float* part) {
    __shared__ float sums[NORM_SUMS][LN_LINES][LN_COLS * VEC + 1];
    const int lane = threadIdx.x % LN_COLS, line = threadIdx.x / LN_COLS;
    const int c = (blockIdx.x * LN_COLS + lane) * VEC;
    float dw[VEC], db[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] = db[j] = 0.f;
    if (c < a.d) {
#pragma unroll 4
        for (long long row = (long long)blockIdx.y * LN_LINES + line; row < a.rows; row += (long long)gridDim.y * LN_LINES) {
            float g[VEC], h[VEC];
            load_some<T, VEC>(static_cast<const T*>(a.dy) + row * a.d + c, g);
            load_some<T, VEC>(static_cast<const T*>(a.h) + row * a.h_stride + c, h);
            const float mean = ln_mean(a, row), rs = a.rstd[row];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                dw[j] = fmaf(g[j], (h[j] - mean) * rs, dw[j]);
                db[j] += g[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        sums[0][line][lane * VEC + j] = dw[j];
        if constexpr (!NORM_RMS) sums[NORM_SUMS - 1][line][lane * VEC + j] = db[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NORM_SUMS * LN_COLS * VEC; i += LN_COLS * LN_LINES) {
        const int which = i / (LN_COLS * VEC), k = i % (LN_COLS * VEC), column = blockIdx.x * LN_COLS * VEC + k;
        if (column >= a.d) continue;
        float s = 0.f;
        for (int l = 0; l < LN_LINES; ++l) s += sums[which][l][k];
        part[((size_t)blockIdx.y * NORM_SUMS + which) * a.d + column] = s;
    }
}

// Sums of the columns of part[parts][NORM_SUMS][d]: LINES threads a column, each with every LINES-th part.
template <class W, int LINES> __global__ void __launch_bounds__(256) ln_columns_finish_kernel(const float* part, int parts, int d, W* dw, W* db) {
    constexpr int COLS = 256 / LINES;
    __shared__ float sums[LINES][COLS];
    const int c = blockIdx.x * COLS + threadIdx.x % COLS, line = threadIdx.x / COLS;
    float s = 0.f;
    if (c < NORM_SUMS * d) {
        const float* p = part + (size_t)line * NORM_SUMS * d + c;
#pragma unroll 8
        for (int i = line; i < parts; i += LINES, p += (size_t)LINES * NORM_SUMS * d) s += *p;
    }
    if constexpr (LINES > 1) {
        sums[line][threadIdx.x % COLS] = s;
        __syncthreads();
        if (line > 0) return;
#pragma unroll
        for (int i = 1; i < LINES; ++i) s += sums[i][threadIdx.x];
    }
    if (c < d) { if (dw != nullptr) dw[c] = from_float<W>(s); }
    else if (!NORM_RMS && c < 2 * d && db != nullptr) db[c - d] = from_float<W>(s);
}

// ------------------------------------------------------------------------------------------ host

// Splits of the rows of the column sums: some 6 CTAs an SM, at least 4 rows a line of a CTA.
int ln_splits(long long rows, int d, int vec) {
    const long long tiles = (d + LN_COLS * vec - 1) / (LN_COLS * vec);
    long long splits = (6LL * sm_count() + tiles - 1) / tiles;
    splits = std::min(splits, (rows + 4 * LN_LINES - 1) / (4 * LN_LINES));
    return (int)std::max(1LL, std::min(splits, 512LL));
}
int ln_most_parts(long long rows) { return (int)std::min(rows, 4LL * sm_count()); }

// CTAs of a kernel that fit on an SM, remembered for each kernel and device.
int resident(const void* kernel, int threads, size_t smem) {
    static std::mutex mu;
    static std::map<std::tuple<const void*, int, size_t>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find({kernel, dev, smem});
    if (it == known.end()) {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) (void)cudaGetLastError();
        it = known.emplace(std::make_tuple(kernel, dev, smem), std::max(n, 1)).first;
    }
    return it->second;
}

// CTAs that share `rows`: as many as are resident, and no more than there are rows for.
template <class S> int ln_ctas(const void* kernel, size_t smem, long long rows) {
    const long long most = std::min(4LL, (long long)resident(kernel, S::THREADS, smem)) * sm_count();
    return (int)std::max(1LL, std::min(most, (rows + S::TEAMS - 1) / S::TEAMS));
}

template <class S, bool EIGHT = false> int launch_forward(const LnFwd& a, int parts, cudaStream_t s) {
    if constexpr (S::STAGES == 0) {
        static_assert(!EIGHT);
        return launch_clusters(ln_forward_row_kernel<S>, (unsigned)((a.rows + S::TEAMS - 1) / S::TEAMS * parts), S::THREADS, 0, parts, s, a);
    } else {
        const auto kernel = ln_forward_kernel<S, EIGHT>;
        const size_t smem = S::ring(a.residual != nullptr ? 2 : 1);
        const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
        if (st != ADDER_OK) return st;
        return launch_clusters(kernel, (unsigned)ln_ctas<S>(reinterpret_cast<const void*>(kernel), smem, a.rows), S::THREADS, smem, 1, s, a);
    }
}

// dx, and with `sums` parts of dw and db: *groups of them are written.
template <class S, bool SUMS> int launch_stay_backward(const LnBwd& a, float* part, int* groups, cudaStream_t s) {
    const auto kernel = ln_backward_kernel<S, SUMS>;
    const size_t teams = SUMS && S::TEAMS > 1 ? (size_t)S::TEAMS * NORM_SUMS * a.d * sizeof(float) : 0;
    const size_t smem = std::max(S::ring(a.dh != nullptr ? 3 : 2), teams);
    const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (st != ADDER_OK) return st;
    *groups = ln_ctas<S>(reinterpret_cast<const void*>(kernel), smem, a.rows);
    return launch_clusters(kernel, (unsigned)*groups, S::THREADS, smem, 1, s, a, part);
}
template <class T, int VEC> int launch_columns(const LnBwd& a, float* part, int* groups, cudaStream_t s) {
    *groups = ln_splits(a.rows, a.d, VEC);
    ln_columns_kernel<T, VEC><<<dim3((unsigned)((a.d + LN_COLS * VEC - 1) / (LN_COLS * VEC)), *groups), LN_COLS * LN_LINES, 0, s>>>(a, part);
    return launched();
}
template <class S> int launch_backward(const LnBwd& a, float* part, bool sums, int parts, int* groups, cudaStream_t s) {
    if constexpr (S::STAGES > 0 || S::THREADS == 512) {
        return sums ? launch_stay_backward<S, true>(a, part, groups, s) : launch_stay_backward<S, false>(a, part, groups, s);
    } else {
        if (a.dx != nullptr) {
            const int st = launch_clusters(ln_dx_row_kernel<S>, (unsigned)(a.rows * parts), S::THREADS, 0, parts, s, a);
            if (st != ADDER_OK) return st;
        }
        return sums ? launch_columns<typename S::T, S::VEC>(a, part, groups, s) : ADDER_OK;
    }
}

constexpr int LN_HELD = 8192;      // columns up to which the backward pass keeps its sums of dw and db from row to row

// Rows beyond 8192 of whole vectors go through shared memory where there are rows for all SMs and two of them fit (2000x20000 bf16: forward 46
// us, backward 105; by clusters 73 and 123); `bytes`: of a row in all arrays that are held.  0: they do not.
size_t wide_bytes(const void* kernel, long long rows, int d, int vec, int ve, size_t bytes) {
    if (d <= LN_HELD || vec != ve || rows < sm_count()) return 0;
    return ensure_dynamic_smem(kernel, 2 * bytes) == ADDER_OK ? 2 * bytes : 0;
}

// f(shape, cluster size) for the shape whose registers hold a row of d elements, in vectors of vec; false: none does.  Whole 16-byte
// vectors go through the ring up to 8192 elements, 16 a thread.  Other rows, and longer ones, which a cluster shares, are held up to 32 a thread
// by CTAs of one row; the backward pass (THREADS = 512) stays where it can, for the sums over the rows.
template <class T, class W, int THREADS, class F> bool with_shape(int d, int vec, F&& f) {
    constexpr int VE = Vec16<T>::N, NV = 16 / VE, STAGES = NV == 2 ? 3 : 2;      // as much shared memory as two CTAs of 256 threads leave
    const auto by_row = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if constexpr (THREADS == 512) {
            if (d <= 128) return f(LnShape<T, W, 32, V, 4 / V, 0, false, 512>(), 1);
            if (d <= 512) return f(LnShape<T, W, 32, V, 16 / V, 0, false, 512>(), 1);
            if (d <= 2048) return f(LnShape<T, W, 128, V, 16 / V, 0, false, 512>(), 1);
            if (d <= LN_HELD) return f(LnShape<T, W, 512, V, 16 / V, 0, false, 512>(), 1);
        } else {
            if (d <= 128) return f(LnShape<T, W, 32, V, 4 / V, 0, false>(), 1);
            if (d <= 512) return f(LnShape<T, W, 32, V, 16 / V, 0, false>(), 1);
            if (d <= 2048) return f(LnShape<T, W, 128, V, 16 / V, 0, false>(), 1);
            if (d <= 4096) return f(LnShape<T, W, 128, V, 32 / V, 0, false>(), 1);
            if (d <= 8192) return f(LnShape<T, W, 256, V, 32 / V, 0, false>(), 1);
        }
        f(LnShape<T, W, 256, V, 32 / V, 0, true>(), (d / V + 256 * (32 / V) - 1) / (256 * (32 / V)));
    };
    if (d > 8 * 8192) return false;
    if (vec == VE) {
        if (d <= 32 * VE) f(LnShape<T, W, 32, VE, 1, 3, false, THREADS>(), 1);
        else if (d <= 512) f(LnShape<T, W, 32, VE, NV, STAGES, false, THREADS>(), 1);
        else if (d <= 1024) f(LnShape<T, W, 64, VE, NV, STAGES, false, THREADS>(), 1);
        else if (d <= 2048) f(LnShape<T, W, 128, VE, NV, STAGES, false, THREADS>(), 1);
        else if (d <= 4096) f(LnShape<T, W, 256, VE, NV, STAGES, false, THREADS>(), 1);
        else if (d <= LN_HELD) f(LnShape<T, W, 512, VE, NV, 2, false, THREADS>(), 1);
        else if (d <= 8 * 4096) f(LnShape<T, W, 256, VE, 16 / VE, 0, true>(), (d / VE + 256 * (16 / VE) - 1) / (256 * (16 / VE)));
        else f(LnShape<T, W, 256, VE, 32 / VE, 0, true>(), (d / VE + 256 * (32 / VE) - 1) / (256 * (32 / VE)));
    } else if (vec == 2) {
        if constexpr (sizeof(T) == 2) by_row(std::integral_constant<int, 2>());
    } else {
        by_row(std::integral_constant<int, 1>());
    }
    return true;
}
// The largest vector that the rows of all tensors allow: 16 bytes, two 16-bit elements, one element.
template <class T> int ln_vector(int d, std::initializer_list<long long> strides, std::initializer_list<const void*> tensors,
                                 std::initializer_list<const void*> weights, unsigned wsize) {
    const auto fits = [&](int vec) {
        if (d % vec != 0) return false;
        for (long long s : strides)
            if (s % vec != 0) return false;
        for (const void* p : tensors)
            if (!aligned_to(p, vec * sizeof(T))) return false;
        for (const void* p : weights)
            if (!aligned_to(p, std::min(16u, vec * wsize))) return false;
        return true;
    };
    return fits(Vec16<T>::N) ? Vec16<T>::N : sizeof(T) == 2 && fits(2) ? 2 : 1;
}
template <class T, class F> int with_weight_type(int wtype, F&& f) {
    if (wtype == ADDER_TYPE_F32) return f(static_cast<float*>(nullptr));
    return f(static_cast<T*>(nullptr));
}

constexpr long long LN_MOST = (1LL << 30) - 65536;      // columns: both sums of all of them are counted in 32 bits

int ln_check(long long rows, long long d, int dtype, int wtype) {
    if (rows < 0 || d <= 0) return ADDER_ERR_BAD_SHAPE;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16 || (wtype != dtype && wtype != ADDER_TYPE_F32)) return ADDER_ERR_UNSUPPORTED;
    if (d > LN_MOST || rows > 2147483647LL / 8) return ADDER_ERR_UNSUPPORTED;
    return ADDER_OK;
}

bool all_aligned(std::initializer_list<const void*> ps, unsigned bytes) {
    for (const void* p : ps)
        if (!aligned_to(p, bytes)) return false;
    return true;
}

// The forward pass of a checked call.
int norm_forward(const LnFwd& a, int dtype, int wtype, cudaStream_t s) {
    const unsigned wsize = wtype == ADDER_TYPE_F32 ? 4 : 2;
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        const int vec = ln_vector<T>(a.d, {a.x_stride, a.residual ? a.r_stride : 0}, {a.x, a.residual, a.y, a.h}, {a.w, a.b}, wsize);
        return with_weight_type<T>(wtype, [&](auto* wt) {
            using W = std::remove_pointer_t<decltype(wt)>;
            int status = ADDER_OK;
            const auto wide = ln_forward_wide_kernel<T, W>;
            const size_t bytes = wide_bytes(reinterpret_cast<const void*>(wide), a.rows, a.d, vec, Vec16<T>::N, a.d * sizeof(T) * (a.residual ? 2 : 1));
            if (bytes > 0) return launch_clusters(wide, (unsigned)sm_count(), LN_WIDE, bytes, 1, s, a);
            const bool held = with_shape<T, W, 256>(a.d, vec, [&](auto shape, int parts) { status = launch_forward<decltype(shape)>(a, parts, s); });
            return held ? status : launch_clusters(ln_forward_long_kernel<T, W>, (unsigned)(a.rows * 8), LN_LONG, 0, 8, s, a);
        });
    });
}

size_t norm_backward_workspace_bytes(long long rows, long long d) {
    if (rows <= 0 || d <= 0 || d > LN_MOST) return 0;
    // Up to LN_HELD columns the CTAs that stay write a part each; beyond, the splits of the pass over the columns do, which are most for
    // the widest vectors.
    const int parts = d <= LN_HELD ? ln_most_parts(rows) : ln_splits(rows, (int)d, 8);
    return (size_t)parts * NORM_SUMS * d * sizeof(float);
}

// The backward pass of a checked call.
int norm_backward(const LnBwd& a, void* dweight, void* dbias, void* workspace, int dtype, int wtype, cudaStream_t s) {
    const unsigned wsize = wtype == ADDER_TYPE_F32 ? 4 : 2;
    const bool sums = dweight != nullptr || dbias != nullptr;
    void* const dx = a.dx;
    const long long d = a.d;
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        const int vec = ln_vector<T>((int)d, {a.h_stride}, {a.dy, a.dh, a.h, dx}, {a.w}, wsize);
        return with_weight_type<T>(wtype, [&](auto* wt) {
            using W = std::remove_pointer_t<decltype(wt)>;
            int status = ADDER_OK, groups = 0;
            float* part = static_cast<float*>(workspace);
            const auto wide = ln_dx_wide_kernel<T, W>;
            const size_t bytes = wide_bytes(reinterpret_cast<const void*>(wide), a.rows, a.d, vec, Vec16<T>::N, d * sizeof(T) * 2);
            const bool held = bytes == 0 && with_shape<T, W, 512>(a.d, vec, [&](auto shape, int parts) {
                status = launch_backward<decltype(shape)>(a, part, sums, parts, &groups, s);
            });
            if (!held) {
                if (dx != nullptr && bytes > 0) status = launch_clusters(wide, (unsigned)sm_count(), LN_WIDE, bytes, 1, s, a);
                else if (dx != nullptr) status = launch_clusters(ln_dx_long_kernel<T, W>, (unsigned)(a.rows * 8), LN_LONG, 0, 8, s, a);
                if (status == ADDER_OK && sums) status = vec == Vec16<T>::N ? launch_columns<T, Vec16<T>::N>(a, part, &groups, s) : launch_columns<T, 1>(a, part, &groups, s);
            }
            if (status != ADDER_OK || !sums) return status;
            // up to 16 parts one after another, more by 16 threads (whole backward pass: 16 parts of 4096 columns 9.3 us and 10.4 by 16; 592 of 1024 12.4
            // one after another and 10.4)
            if (groups <= 16) ln_columns_finish_kernel<W, 1><<<(unsigned)((NORM_SUMS * d + 255) / 256), 256, 0, s>>>(part, groups, a.d, static_cast<W*>(dweight), static_cast<W*>(dbias));
            else ln_columns_finish_kernel<W, 16><<<(unsigned)((NORM_SUMS * d + 15) / 16), 256, 0, s>>>(part, groups, a.d, static_cast<W*>(dweight), static_cast<W*>(dbias));
            return launched();
        });
    });
}

}  // namespace
}  // namespace adder
