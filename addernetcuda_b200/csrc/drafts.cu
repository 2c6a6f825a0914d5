// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   a sequence has L drafted tokens t_i, each drawn from probabilities q_i, and the target's probabilities p_0 .. p_L
//   n = the first i with not (u_i q_i(t_i) < p_i(t_i)), or L;  then one more token, of weights w(c):
//     max(p_n(c) - q_n(c), 0) where n < L (p_n(c), without t_n, where the drafter gives no probabilities), or p_L(c) where n = L
//   token = the first c with sum_{c' <= c} w(c') > u sum w  and  w(c) > 0
//
// The sums are held in 64 bits: differences of two values are exact there, and a border between two classes moves by some 1e-16 of the whole,
// so the token does not depend on the order of a sum in practice (in 32 bits it would, for one draw in a hundred of 128000 classes).
//
// A sequence's row is split over a cluster of CTAs and their warps, a segment of consecutive classes a warp.  Every CTA finds n for itself,
// sums its segments and leaves the sums with all CTAs of the cluster; then the CTA whose segment holds the border reads that again, a part a warp.
//
// What bounds it: of all rows only those of p_n and q_n are read, in lines that nothing has touched before, behind three loads that wait for one
// another (the tokens, their probabilities, the row), and the segment's second reading waits for the sums.  One sequence of 32000 fp32 classes 6.4 us;
// 64 of 128000 bf16 14.3 us, where the bytes alone take 5 (with 512 threads a CTA or 256, and with additions in fp32 instead of 64 bits, the same).
#include "kernels.h"
#include "elements.cuh"
#include "launch.cuh"
#include <cooperative_groups.h>

namespace adder {
namespace {

namespace cg = cooperative_groups;

constexpr int DV_THREADS = 512, DV_WARPS = DV_THREADS / 32, DV_MOST_PARTS = 8;
constexpr int DV_EACH = DV_MOST_PARTS * DV_WARPS / 32;      // segments a lane

struct DvArgs {
    const void* p;                 // [sequences][drafts + 1][classes]
    const void* q;                 // [sequences][drafts][classes], or null: the drafter is certain of its tokens
    const long long* tokens;       // [sequences][drafts]
    const float* u;                // [sequences][drafts + 1]
    const long long* lengths;      // [sequences], or null
    long long* out;                // [sequences][drafts + 1]
    long long* accepted;           // [sequences]
    long long p_sequence, p_place, q_sequence, q_place;      // strides
    int drafts, classes;
};

template <class T, int N> __device__ __forceinline__ void dv_load(const T* p, float (&f)[N]) {
    if constexpr (N == 1) f[0] = to_float(*p);
    else Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
// Weights below fp32's smallest normal number count as nothing, NaN too.
constexpr float DV_LEAST = 0x1p-126f;
// A weight of at least that in 64 bits, by its bits: a conversion takes 16 clocks of a scheduler (64x6x128000 20.6 us with them).  Infinity becomes 2^128.
__device__ __forceinline__ double dv_double(float w) {
    const uint32_t u = __float_as_uint(w);
    return __hiloint2double((int)((u >> 3) + 0x38000000u), (int)(u << 29));
}
// f - g, and what fp32 leaves out of it.  The operations after d are exact as long as nothing overflows.
__device__ __forceinline__ float dv_difference(float f, float g, float& left) {
    const float d = f - g, b = d - f;
    const float e = (f - (d - b)) - (g + b);
    left = d >= DV_LEAST && d < INFINITY ? e : 0.f;
    return d;
}
// Differences of values in 16 bits, of which nothing is left out but where one is some 2^16 (bf16) or 2^13 (fp16) times the other: `far` stays 0 but
// then.  For d > 0 and g >= 0 g + (d - f) is minus what is left out, exactly; where g is negative nothing is said.
template <int VEC> __device__ __forceinline__ void dv_differences(const float (&f)[VEC], const float (&g)[VEC], float (&d)[VEC], uint32_t& far) {
    if constexpr (VEC == 1) {
        d[0] = f[0] - g[0];
        far |= __float_as_uint(g[0] + (d[0] - f[0])) | (__float_as_uint(g[0]) & 0x80000000u);
    } else {
        const uint64_t minus = pack2(-1.f, -1.f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const uint64_t f2 = pack2(f[j], f[j + 1]), g2 = pack2(g[j], g[j + 1]), d2 = fma2(g2, minus, f2);
            float lo, hi;
            unpack2(add2(g2, fma2(f2, minus, d2)), lo, hi);
            unpack2(d2, d[j], d[j + 1]);
            far |= __float_as_uint(lo) | __float_as_uint(hi) | ((__float_as_uint(g[j]) | __float_as_uint(g[j + 1])) & 0x80000000u);
        }
    }
}
// Inclusive sums over the lanes of a warp.
__device__ __forceinline__ double dv_scan(double v, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// VEC consecutive classes a lane at a time.
template <class T, int VEC> __global__ void __launch_bounds__(DV_THREADS) dv_kernel(const DvArgs a) {
    __shared__ double sums[2][DV_MOST_PARTS * DV_WARPS];
    __shared__ double part_of[DV_WARPS];
    __shared__ int first_refused;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const long long b = blockIdx.x / parts;
    const long long* tokens = a.tokens + b * a.drafts;
    const float* u = a.u + b * (a.drafts + 1);
    const T* p = static_cast<const T*>(a.p) + b * a.p_sequence;
    const T* q = a.q != nullptr ? static_cast<const T*>(a.q) + b * a.q_sequence : nullptr;
    const int length = a.lengths == nullptr ? a.drafts : (int)max(0LL, min((long long)a.drafts, a.lengths[b]));

    const float u_last = u[a.drafts];
    if (warp == 0) {
        int n = length;
        for (int base = 0; base < length; base += 32) {
            const int i = base + lane;
            bool stands = true;
            if (i < length) {
                const long long token = tokens[i];
                stands = false;      // what is no class does not stand
                if (token >= 0 && token < a.classes) {
                    const double pt = to_float(p[i * a.p_place + token]), qt = q == nullptr ? 1.0 : (double)to_float(q[i * a.q_place + token]);
                    stands = (double)u[i] * qt < pt;
                }
            }
            const unsigned refused = ~__ballot_sync(0xffffffffu, stands);
            if (refused != 0) {
                n = base + __ffs(refused) - 1;
                break;
            }
        }
        if (lane == 0) first_refused = n;
    }
    __syncthreads();
    const int n = first_refused;
    const T* p_row = p + n * a.p_place;
    const T* q_row = n < length && q != nullptr ? q + n * a.q_place : nullptr;
    const int gone = n < length && q == nullptr && tokens[n] >= 0 && tokens[n] < a.classes ? (int)tokens[n] : -1;
    const int segments = parts * DV_WARPS, segment = rank * DV_WARPS + warp, nvec = a.classes / VEC, shift = 31 - __clz(segments);      // a power of two
    const auto segment_begin = [&](int i) { return (int)((long long)nvec * i >> shift); };
    const int v0 = segment_begin(segment), v1 = segment_begin(segment + 1);

    // Weights of the classes of vector v, and what fp32 leaves out of them; with `whole` those of p alone.
    const auto weights = [&](int v, bool whole, float (&w)[VEC], float (&left)[VEC]) {
        float f[VEC];
        dv_load<T, VEC>(p_row + (size_t)v * VEC, f);
        if (q_row == nullptr || whole) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                w[j] = !whole && v * VEC + j == gone ? 0.f : f[j];
                left[j] = 0.f;
            }
        } else {
            float g[VEC];
            dv_load<T, VEC>(q_row + (size_t)v * VEC, g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[j] = dv_difference(f[j], g[j], left[j]);
        }
    };
    // Sum of the weights of vectors from to to - 1, in every lane of a warp.  In 16 bits what is left out of differences is asked for, and a lane that has
    // any goes over its vectors again for it (64x6x128000 bf16 14.3 us; added up beside every difference 22, by a branch at
    // each vector 20.5).
    const auto sum_of = [&](int from, int to, bool whole) {
        double sum[2] = {0.0, 0.0};
        float rest = 0.f;
        if (sizeof(T) == 4 || q_row == nullptr || whole) {
#pragma unroll 4
            for (int v = from + lane; v < to; v += 32) {
                float w[VEC], left[VEC];
                weights(v, whole, w, left);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (w[j] >= DV_LEAST) sum[j & 1] += dv_double(w[j]);
                    rest += left[j];
                }
            }
        } else {
            uint32_t far = 0;
#pragma unroll 4
            for (int v = from + lane; v < to; v += 32) {
                float f[VEC], g[VEC], w[VEC];
                dv_load<T, VEC>(p_row + (size_t)v * VEC, f);
                dv_load<T, VEC>(q_row + (size_t)v * VEC, g);
                dv_differences<VEC>(f, g, w, far);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (w[j] >= DV_LEAST) sum[j & 1] += dv_double(w[j]);
            }
            if (far != 0) {
#pragma unroll 1
                for (int v = from + lane; v < to; v += 32) {
                    float w[VEC], left[VEC];
                    weights(v, false, w, left);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) rest += left[j];
                }
            }
        }
        double s = sum[0] + sum[1] + (double)rest;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        return s;
    };
    // Sums of all segments in the lanes of every warp, DV_EACH a lane: what lies before them, and theirs.
    double before = 0.0, mine[DV_EACH], total = 0.0;
    const auto sum_up = [&](bool whole, int turn) {
        const double s = sum_of(v0, v1, whole);
        if (turn == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // all CTAs of the cluster have begun
        if (lane < parts) cluster.map_shared_rank(&sums[turn][0], lane)[segment] = s;
        cluster.sync();
        double own = 0.0;
#pragma unroll
        for (int i = 0; i < DV_EACH; ++i) {
            mine[i] = DV_EACH * lane + i < segments ? sums[turn][DV_EACH * lane + i] : 0.0;
            own += mine[i];
        }
        const double all = dv_scan(own, lane);
        before = __shfl_up_sync(0xffffffffu, all, 1);
        if (lane == 0) before = 0.0;
        total = __shfl_sync(0xffffffffu, all, 31);
    };
    sum_up(false, 0);
    bool whole = false;
    if (total == 0.0) {      // p nowhere above q: rounding alone, or probabilities that are none
        whole = true;
        sum_up(true, 1);
    }
    const double want = (double)u_last * total;
    if (rank == 0) {
        for (int i = t; i <= a.drafts; i += DV_THREADS) {
            if (i < n) a.out[b * (a.drafts + 1) + i] = tokens[i];
            else if (i > n) a.out[b * (a.drafts + 1) + i] = -1;
        }
        if (t == 0) a.accepted[b] = n;
    }
    if (!(total > 0.0) || total >= 0x1p128) {      // no class has a weight, or one has no finite one
        if (rank == 0 && t == 0) a.out[b * (a.drafts + 1) + n] = -1;
        return;
    }
    // The segment that holds the border, or, where rounding or u >= 1 leaves none, the last with a weight; and what lies before it.
    double reached = before, before_last = before;
    int holds = -1, some = -1;
#pragma unroll
    for (int i = 0; i < DV_EACH; ++i) {
        if (mine[i] > 0.0 && holds < 0) {
            some = i;
            before_last = reached;
            if (reached + mine[i] > want) holds = i;
        }
        reached += mine[i];
    }
    const unsigned holders = __ballot_sync(0xffffffffu, holds >= 0), weighty = __ballot_sync(0xffffffffu, some >= 0);
    const int from_lane = holders != 0 ? __ffs(holders) - 1 : 31 - __clz(weighty);
    const int chosen = DV_EACH * from_lane + __shfl_sync(0xffffffffu, some, from_lane);      // the holding one where there is one
    reached = __shfl_sync(0xffffffffu, before_last, from_lane);
    // Its CTA reads the segment again, a part a warp and consecutive vectors a lane; the lane whose vectors hold the border (or the last weight) goes
    // over them once more.
    if (chosen / DV_WARPS != rank) return;
    const int c0 = segment_begin(chosen), c1 = segment_begin(chosen + 1);
    const int p0 = c0 + (int)((long long)(c1 - c0) * warp / DV_WARPS), p1 = c0 + (int)((long long)(c1 - c0) * (warp + 1) / DV_WARPS), each = (p1 - p0 + 31) / 32;
    const int l0 = min(p1, p0 + lane * each), l1 = min(p1, l0 + each);
    double own = 0.0;
    for (int v = l0; v < l1; ++v) {
        float w[VEC], left[VEC];
        weights(v, whole, w, left);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (w[j] >= DV_LEAST) own += dv_double(w[j]) + (double)left[j];
    }
    const double upto = dv_scan(own, lane);
    if (lane == 31) part_of[warp] = upto;
    __syncthreads();
    const double mass = lane < DV_WARPS ? part_of[lane] : 0.0, end = reached + dv_scan(mass, lane);
    const unsigned hold = __ballot_sync(0xffffffffu, mass > 0.0 && end > want), any = __ballot_sync(0xffffffffu, mass > 0.0);
    const int part = hold != 0 ? __ffs(hold) - 1 : 31 - __clz(any);
    reached = __shfl_sync(0xffffffffu, end - mass, part);
    if (warp != part) return;
    const unsigned hold_lane = __ballot_sync(0xffffffffu, own > 0.0 && reached + upto > want), any_lane = __ballot_sync(0xffffffffu, own > 0.0);
    if (lane != (hold_lane != 0 ? __ffs(hold_lane) - 1 : 31 - __clz(any_lane))) return;
    double at = reached + (upto - own);
    int token = -1;
    for (int v = l0; v < l1 && !(at > want && token >= 0); ++v) {
        float w[VEC], left[VEC];
        weights(v, whole, w, left);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (w[j] >= DV_LEAST && !(at > want && token >= 0)) {
                at += dv_double(w[j]) + (double)left[j];
                token = v * VEC + j;
            }
    }
    a.out[b * (a.drafts + 1) + n] = token;
}

template <class T, int VEC> int launch_drafts(const DvArgs& a, long long sequences, cudaStream_t s) {
    // A CTA takes at least some 2048 classes, and there are up to two an SM.
    int parts = 1;
    while (parts < DV_MOST_PARTS && a.classes >= 4096LL * parts && sequences * parts * 2 <= 2LL * sm_count()) parts *= 2;
    return launch_clusters(dv_kernel<T, VEC>, (unsigned)(sequences * parts), DV_THREADS, 0, parts, s, a);
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" int adder_b200_verify_drafts(const void* target, const void* draft, int dtype, const long long* tokens, const float* uniforms,
                                        const long long* lengths, long long* out_tokens, long long* accepted, long long sequences, long long drafts,
                                        long long classes, long long target_sequence_stride, long long target_place_stride,
                                        long long draft_sequence_stride, long long draft_place_stride, void* stream) {
    if (sequences < 0 || drafts < 0 || classes <= 0) return ADDER_ERR_BAD_SHAPE;
    if (target_sequence_stride < 0 || target_place_stride < 0 || draft_sequence_stride < 0 || draft_place_stride < 0) return ADDER_ERR_BAD_SHAPE;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16) return ADDER_ERR_UNSUPPORTED;
    if (classes > 2147483647LL - 1024 || drafts > 65535 || sequences > 2147483647LL / DV_MOST_PARTS) return ADDER_ERR_UNSUPPORTED;
    if (sequences == 0) return ADDER_OK;
    if (!target || !uniforms || !out_tokens || !accepted || (drafts > 0 && !tokens)) return ADDER_ERR_NULL_POINTER;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!aligned_to(target, size) || !aligned_to(draft, size) || !aligned_to(tokens, 8) || !aligned_to(lengths, 8) || !aligned_to(out_tokens, 8) ||
        !aligned_to(accepted, 8) || !aligned_to(uniforms, 4))
        return ADDER_ERR_ALIGNMENT;
    const DvArgs a{target, draft, tokens, uniforms, lengths, out_tokens, accepted, target_sequence_stride, target_place_stride,
                   draft_sequence_stride, draft_place_stride, (int)drafts, (int)classes};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int VE = Vec16<T>::N;
        bool vectors = classes % VE == 0 && aligned_to(target, 16) && aligned_to(draft, 16);
        for (long long stride : {target_sequence_stride, target_place_stride, draft_sequence_stride, draft_place_stride}) vectors = vectors && stride % VE == 0;
        return vectors ? launch_drafts<T, VE>(a, sequences, s) : launch_drafts<T, 1>(a, sequences, s);
    });
}
