// Distillation from a teacher's top logits: how far a row's softmax is from the teacher's, and its gradient.
//
//   forward   t = softmax(z / T) over the k classes i_j that the teacher names, p = softmax(x / T), M = max x
//             D = sum_j t_j (ln t_j - ln p_{i_j}),  ln p_i = (x_i - M) / T - ln sum e^((x - M) / T);  log softmax(x) at a target class
//   backward  dx_i = g_D / T (p_i - sum_{j: i_j = i} t_j) + g_L ([i = target] - softmax(x)_i)
//
// The forward reads the logits once: every thread keeps a maximum of its own with the sums relative to it (two where the target's
// probability at temperature 1 is asked for beside another temperature), which are rescaled when it rises and joined at the end.  It leaves M,
// the sums and t for the backward, which reads the logits again and writes the gradient.
//
// What bounds it: memory (2048x128000 bf16: forward 89 us, 90 % of a copy's rate, with the label's probability at T = 2 or 4 96 us; backward 165 us,
// 97 %), the exponential unit where two exponentials are taken (T = 3 with labels 149 us), and a row's beginning and end in shorter ones (2048x50257
// with 64 classes of the teacher's 44 us, 71 %).  256x1000 fp32, a warp a row, waits for its loads: 6.8 us forward, 6.8 backward.  Where the gradient's rows
// lie otherwise on 16 bytes than the logits', the backward goes element by element: 2048x50257 in rows of 50304 275 us bf16 and 291 fp32, dense rows 88
// and 142.
#include "kernels.h"
#include "launch.cuh"
#include "logit_rows.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace adder {
namespace {

namespace cg = cooperative_groups;

constexpr int DS_MAX_K = 256, DS_TEAM = LP_TEAM;
constexpr int DS_UNROLL = 4;            // backward: vectors that a thread has in flight

struct DsFwd {
    const void* x;
    long long rows, stride;
    int classes, k;
    const void* teacher;             // [rows][k]
    int teacher_type;
    const long long* indices;        // [rows][k]
    const long long* targets;        // [rows], or null
    long long ignore;
    float inv_t;                     // 1 / T
    float scale;                     // log2(e) / T
    float* divergence;               // [rows]
    float* log_prob;                 // [rows], with targets
    float* stats;                    // [rows][3]: M and both sums; or null
    float* mass;                     // [rows][k]: t; or null
};

// What a row's second sum, at temperature 1, is made of: nothing (ONE: none is asked for, or the temperature is 1), an exponential of its own
// (OWN), or the first one's squared (SQUARE: T = 2) or its fourth power (FOURTH: T = 4).  The exponential unit takes 8 clocks of a scheduler for a
// warp's values and memory 11, so a second exponential costs time and two products do not (2048x128000 bf16: 145 us with OWN).
enum DsSecond { ONE, OWN, SQUARE, FOURTH };
template <int SECOND> __device__ __forceinline__ uint64_t ds_second(uint64_t d, uint64_t e) {
    if constexpr (SECOND == OWN) {
        float lo, hi;
        unpack2(mul2(d, pack2(LOG2E, LOG2E)), lo, hi);
        return pack2(exp2_fast(lo), exp2_fast(hi));
    } else {
        const uint64_t square = mul2(e, e);
        return SECOND == SQUARE ? square : mul2(square, square);
    }
}

// Largest value m with sums of 2^((x - m) scale) and, but with ONE, of 2^((x - m) log2 e).
template <int SECOND> struct DsSums {
    float m = -INFINITY;
    uint64_t s = 0, s1 = 0;      // pairs

    __device__ __forceinline__ void raise(float top, float scale) {
        const float f = m == -INFINITY ? 0.f : exp2_fast((m - top) * scale);
        s = mul2(s, pack2(f, f));
        if (SECOND != ONE) {
            const float f1 = m == -INFINITY ? 0.f : exp2_fast((m - top) * LOG2E);
            s1 = mul2(s1, pack2(f1, f1));
        }
        m = top;
    }
    __device__ __forceinline__ void add(float a, float b, float scale) {
        const uint64_t d = add2(pack2(a, b), pack2(-m, -m));
        float lo, hi;
        unpack2(mul2(d, pack2(scale, scale)), lo, hi);
        const uint64_t e = pack2(exp2_fast(lo), exp2_fast(hi));
        s = add2(s, e);
        if constexpr (SECOND != ONE) s1 = add2(s1, ds_second<SECOND>(d, e));
    }
};
struct DsPart {
    float m, s, s1;
};
// Sums relative to the larger maximum.  Equal maxima (both -inf among them) need no factor; a NaN stays one.
__device__ __forceinline__ DsPart ds_join(DsPart a, DsPart b, float scale) {
    const float m = max_nan(a.m, b.m);
    const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
    return {m, a.s * exp2_fast(da * scale) + b.s * exp2_fast(db * scale), a.s1 * exp2_fast(da * LOG2E) + b.s1 * exp2_fast(db * LOG2E)};
}
__device__ __forceinline__ DsPart ds_join_lanes(DsPart p, float scale) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const DsPart o{__shfl_xor_sync(0xffffffffu, p.m, off), __shfl_xor_sync(0xffffffffu, p.s, off), __shfl_xor_sync(0xffffffffu, p.s1, off)};
        p = ds_join(p, o, scale);
    }
    return p;
}

// Values of a vector into the sums.
template <class T, int U, int SECOND> __device__ __forceinline__ void ds_take(const uint4 (&q)[U], DsSums<SECOND>& run, float scale) {
    constexpr int VE = Vec16<T>::N;
    uint32_t w;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t a = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
        w = u == 0 ? a : max_word<T>(w, a);
    }
    const float top = word_max<T>(w);
    if (top > run.m || top != top) run.raise(top, scale);      // a NaN stays
    if (run.m == -INFINITY) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float f[VE];
        Vec16<T>::unpack(q[u], f);
#pragma unroll
        for (int i = 0; i < VE; i += 2) run.add(f[i], f[i + 1], scale);
    }
}

__device__ __forceinline__ float ds_value(const void* p, int type, long long i) {
    if (type == ADDER_TYPE_F32) return static_cast<const float*>(p)[i];
    return type == ADDER_TYPE_BF16 ? to_float(static_cast<const __nv_bfloat16*>(p)[i]) : to_float(static_cast<const __half*>(p)[i]);
}

// The sums of a row's share of a thread, every THREADS-th vector, on their way through shared memory (double-buffered in registers instead, the forward
// of 2048x128000 bf16 took 104 us).
template <class T, int THREADS, int SECOND> struct DsReader {
    using Stream = LpStream<T, THREADS>;
    Stream stream;
    uint32_t from;

    __device__ __forceinline__ void begin(const DsFwd& a, uint4* ring, long long row, long long step, int t, int rank, int parts) {
        stream.first = stream.at = from = smem_u32(ring) + threadIdx.x * 16;
        stream.row = row;
        stream.step = step;
        stream.set_row(a, t, rank, parts);
#pragma unroll
        for (int i = 0; i < LP_STAGES - 1; ++i) stream.issue(a, t, rank, parts);
    }
    __device__ __forceinline__ DsPart read(const DsFwd& a, const LpRow<T>& r, int t, int rank, int parts) {
        const float one = t < r.singles ? to_float(r.x[r.single(t)]) : -INFINITY;
        DsSums<SECOND> run;
        int v = r.v0 + t;
        for (int g = r.groups(THREADS); g > 0; --g) {
            stream.issue(a, t, rank, parts);
            cp_async_wait<LP_STAGES - 1>();
            if (v + (LP_GROUP - 1) * THREADS < r.v1) {
                uint4 q[LP_GROUP];
#pragma unroll
                for (int u = 0; u < LP_GROUP; ++u) q[u] = read16(from + u * Stream::SLOT);
                ds_take<T, LP_GROUP>(q, run, a.scale);
            } else {
#pragma unroll 1
                for (int u = 0; u < LP_GROUP - 1 && v + u * THREADS < r.v1; ++u) {
                    const uint4 q[1] = {read16(from + u * Stream::SLOT)};
                    ds_take<T, 1>(q, run, a.scale);
                }
            }
            from = from == stream.first + Stream::RING - Stream::STAGE ? stream.first : from + Stream::STAGE;
            v += LP_GROUP * THREADS;
        }
        if (one > run.m || one != one) run.raise(one, a.scale);
        if (t < r.singles && run.m != -INFINITY) run.add(one, -INFINITY, a.scale);
        float lo, hi, lo1, hi1;
        unpack2(run.s, lo, hi);
        unpack2(run.s1, lo1, hi1);
        return {run.m, lo + hi, lo1 + hi1};
    }
};

// What the teacher says of a row, looked up by a warp: its classes' logits by the teacher and of the row, their indices (-1: none), and the target.
struct DsNamed {
    float z[DS_MAX_K], x[DS_MAX_K];
    int at[DS_MAX_K];
};
template <class T> struct DsTold {
    bool broken;
    long long target;
    float x_target;

    __device__ __forceinline__ void look_up(const DsFwd& a, long long row, const T* x, int lane, DsNamed& named) {
        broken = false;
        target = a.targets != nullptr ? a.targets[row] : a.ignore;
        for (int j = lane; j < a.k; j += 32) {
            const long long i = a.indices[row * a.k + j];
            broken |= i >= a.classes || i < -1;
            const bool in = i >= 0 && i < a.classes;
            named.at[j] = in ? (int)i : -1;
            named.z[j] = ds_value(a.teacher, a.teacher_type, row * a.k + j);
            broken |= named.z[j] != named.z[j];      // at an empty place, too: log probabilities name no class in a row that has failed
            if (in) named.x[j] = to_float(x[i]);
        }
        x_target = target >= 0 && target < a.classes ? to_float(x[target]) : 0.f;
        broken = __any_sync(0xffffffffu, broken);
        __syncwarp();
    }
};

// A row's outputs from its sums, by the warp that has looked up what the teacher says.
template <class T, int SECOND> __device__ __forceinline__ void ds_finish(const DsFwd& a, long long row, const DsPart& all, const DsTold<T>& told, const DsNamed& named, int lane) {
    float top = -INFINITY;
    for (int j = lane; j < a.k; j += 32)
        if (named.at[j] >= 0) top = max_nan(top, named.z[j]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    const bool broken = told.broken || top == INFINITY || top != top, empty = top == -INFINITY;
    float sum = 0.f;
    for (int j = lane; j < a.k; j += 32)
        if (named.at[j] >= 0 && !empty) sum += exp2_fast((named.z[j] - top) * a.scale);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float log_mass = logf(sum), log_sum = logf(all.s);
    float d = 0.f;
    for (int j = lane; j < a.k; j += 32) {
        float share = 0.f;
        if (named.at[j] >= 0 && !empty) {
            const float e = (named.z[j] - top) * a.inv_t;
            share = exp2_fast((named.z[j] - top) * a.scale) / sum;
            if (share > 0.f) d += share * (e - log_mass - ((named.x[j] - all.m) * a.inv_t - log_sum));
        }
        if (a.mass != nullptr) a.mass[row * a.k + j] = broken ? NAN : share;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
    if (lane == 0) {
        const bool nothing = all.m == -INFINITY;
        const float s1 = SECOND != ONE ? all.s1 : all.s;
        a.divergence[row] = broken ? NAN : empty ? 0.f : nothing ? INFINITY : d;
        if (a.targets != nullptr)
            a.log_prob[row] = told.target == a.ignore ? 0.f : told.target < 0 || told.target >= a.classes ? NAN : nothing ? -INFINITY : told.x_target - all.m - logf(s1);
        if (a.stats != nullptr) {
            a.stats[3 * row] = all.m;
            a.stats[3 * row + 1] = all.s;
            a.stats[3 * row + 2] = s1;
        }
    }
}

// A warp a row, four of them a CTA.
template <class T, int SECOND> __global__ void __launch_bounds__(128) ds_warp_kernel(const DsFwd a) {
    extern __shared__ uint4 ring[];
    __shared__ DsNamed named_of[4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= a.rows) return;
    LpRow<T> r;
    r.set(a, row, 0, 1);
    DsReader<T, 32, SECOND> reader;
    reader.begin(a, ring, row, a.rows, lane, 0, 1);
    DsTold<T> told;
    told.look_up(a, row, r.x, lane, named_of[warp]);
    ds_finish<T, SECOND>(a, row, ds_join_lanes(reader.read(a, r, lane, 0, 1), a.scale), told, named_of[warp], lane);
}

// A CTA's rows one after another: DS_TEAM threads read them, and a warp more finishes each while the others read the next (2048x50257 bf16 with 64 classes
// of the teacher's: 47 us where a CTA of DS_TEAM threads did one row and all of it).
constexpr int DS_STREAM = DS_TEAM + 32;
enum { DS_EMPTY = 1, DS_FULL = 3 };      // named barriers, two of each; 0 is __syncthreads
__device__ __forceinline__ void ds_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(DS_STREAM) : "memory"); }
__device__ __forceinline__ void ds_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(DS_STREAM) : "memory"); }

template <class T, int SECOND> __global__ void __launch_bounds__(DS_STREAM, 4) ds_stream_kernel(const DsFwd a) {
    constexpr int WARPS = DS_TEAM / 32;
    extern __shared__ uint4 ring[];
    __shared__ DsPart parts_of[2][WARPS];
    __shared__ DsNamed named;
    const int t = threadIdx.x, lane = t & 31;
    long long row = blockIdx.x;
    LpRow<T> r;
    if (t < DS_TEAM) {
        DsReader<T, DS_TEAM, SECOND> reader;
        reader.begin(a, ring, row, gridDim.x, t, 0, 1);
        for (int turn = 0; row < a.rows; turn ^= 1, row += gridDim.x) {
            r.set(a, row, 0, 1);
            const DsPart mine = ds_join_lanes(reader.read(a, r, t, 0, 1), a.scale);
            ds_sync(DS_EMPTY + turn);      // the row before the last is finished
            if (lane == 0) parts_of[turn][t >> 5] = mine;
            __syncwarp();
            ds_arrive(DS_FULL + turn);
        }
        return;
    }
    ds_arrive(DS_EMPTY);
    if (row + gridDim.x < a.rows) ds_arrive(DS_EMPTY + 1);      // where there is one row, nobody waits for this
    for (int turn = 0; row < a.rows; turn ^= 1, row += gridDim.x) {
        r.set(a, row, 0, 1);
        DsTold<T> told;
        told.look_up(a, row, r.x, lane, named);
        ds_sync(DS_FULL + turn);
        const DsPart all = lane < WARPS ? parts_of[turn][lane] : DsPart{-INFINITY, 0.f, 0.f};
        __syncwarp();
        // those that will wait for it: the rows after the next
        if (row + 2 * (long long)gridDim.x < a.rows) ds_arrive(DS_EMPTY + turn);
        ds_finish<T, SECOND>(a, row, ds_join_lanes(all, a.scale), told, named, lane);
        __syncwarp();
    }
}

// Few rows: each is shared out over a cluster of CTAs.
template <class T, int SECOND> __global__ void __launch_bounds__(DS_TEAM) ds_cluster_kernel(const DsFwd a) {
    constexpr int WARPS = DS_TEAM / 32;
    extern __shared__ uint4 ring[];
    __shared__ DsPart parts_of[WARPS], ranks_of[8];
    __shared__ DsNamed named;
    const int t = threadIdx.x, lane = t & 31, parts = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const long long row = blockIdx.x / parts;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    LpRow<T> r;
    r.set(a, row, rank, parts);
    DsReader<T, DS_TEAM, SECOND> reader;
    reader.begin(a, ring, row, a.rows, t, rank, parts);
    DsTold<T> told;
    if (rank == 0 && t < 32) told.look_up(a, row, r.x, lane, named);
    const DsPart mine = ds_join_lanes(reader.read(a, r, t, rank, parts), a.scale);
    if (lane == 0) parts_of[t >> 5] = mine;
    __syncthreads();
    DsPart all = lane < WARPS ? parts_of[lane] : DsPart{-INFINITY, 0.f, 0.f};
    all = ds_join_lanes(all, a.scale);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // all CTAs of the cluster have begun
    if (t == 0) cg::this_cluster().map_shared_rank(ranks_of, 0)[rank] = all;
    cg::this_cluster().sync();
    if (rank != 0 || t >= 32) return;
    all = lane < parts ? ranks_of[lane] : DsPart{-INFINITY, 0.f, 0.f};
    ds_finish<T, SECOND>(a, row, ds_join_lanes(all, a.scale), told, named, lane);
}

struct DsBwd {
    const void* x;
    long long rows, stride;
    int classes, k;
    const long long* indices;
    const long long* targets;        // or null
    long long ignore;
    float inv_t, scale;
    const float* stats;
    const float* mass;
    const float* g_divergence;       // [rows], or null
    const float* g_log_prob;         // [rows], or null
    void* dx;
    int segments;                    // of a row
};

// What a row's elements have in common: dx = soft 2^((x - m) scale) + hard 2^((x - m) log2 e)
template <int SECOND> struct DsSlope {
    float m, soft, hard, scale;
    __device__ __forceinline__ uint64_t pair(float a, float b) const {
        const uint64_t d = add2(pack2(a, b), pack2(-m, -m));
        float lo, hi;
        unpack2(mul2(d, pack2(scale, scale)), lo, hi);
        const uint64_t e = pack2(exp2_fast(lo), exp2_fast(hi));
        const uint64_t r = mul2(e, pack2(soft, soft));
        if constexpr (SECOND != ONE) return fma2(ds_second<SECOND>(d, e), pack2(hard, hard), r);
        else return r;
    }
    __device__ __forceinline__ float one(float a) const {
        float lo, hi;
        unpack2(pair(a, a), lo, hi);
        return lo;
    }
};

template <class T, int THREADS, int SECOND> __global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) ds_backward_kernel(const DsBwd a) {
    constexpr int VE = Vec16<T>::N;
    const int t = threadIdx.x % THREADS;
    // from the last row on: what the forward read last is still in L2
    const long long row = a.rows - 1 - (THREADS == 32 ? (long long)blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x / a.segments);
    const int segment = THREADS == 32 ? 0 : (int)(blockIdx.x % a.segments);
    if (row < 0) return;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* dx = static_cast<T*>(a.dx) + row * (long long)a.classes;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const bool same = (reinterpret_cast<uintptr_t>(dx) & 15) == (reinterpret_cast<uintptr_t>(x) & 15);
    const int head = min(a.classes, mis == 0 ? 0 : VE - mis), nvec = (a.classes - head) / VE;
    const int v0 = (int)((long long)nvec * segment / a.segments), v1 = (int)((long long)nvec * (segment + 1) / a.segments);
    const uint4* vec = reinterpret_cast<const uint4*>(x + head);
    uint4 q[DS_UNROLL];
    if (same) {      // on their way while the row's numbers are looked up
#pragma unroll
        for (int u = 0; u < DS_UNROLL; ++u)
            if (v0 + t + u * THREADS < v1) q[u] = __ldg(vec + v0 + t + u * THREADS);
    }
    const float m = a.stats[3 * row], s = a.stats[3 * row + 1], s1 = a.stats[3 * row + 2];
    const bool nothing = m == -INFINITY;
    const float gd = a.g_divergence != nullptr ? a.g_divergence[row] * a.inv_t : 0.f;
    const long long target = a.targets != nullptr && a.g_log_prob != nullptr ? a.targets[row] : a.ignore;
    const float gl = target == a.ignore ? 0.f : target < 0 || target >= a.classes ? NAN : a.g_log_prob[row];
    // A row without classes of the teacher's has no part of the divergence, nor has one whose divergence has no gradient (a row that is ignored), whatever
    // the teacher says of it; one with a NaN among its shares is NaN.
    const float* mass = a.mass + row * a.k;
    const long long* at = a.indices + row * a.k;
    float some = 0.f;
    for (int j = threadIdx.x & 31; j < a.k; j += 32) some = max_nan(some, mass[j]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) some = max_nan(some, __shfl_xor_sync(0xffffffffu, some, off));
    DsSlope<SECOND> slope;
    slope.m = m;
    slope.scale = a.scale;
    const float soft = some == 0.f || gd == 0.f ? 0.f : some != some ? NAN : gd;
    slope.soft = soft / s;
    slope.hard = -gl / s1;
    if (SECOND == ONE) slope.soft += slope.hard;

    int begin, end;
    if (same) {
        uint4* out = reinterpret_cast<uint4*>(dx + head);
        for (int v = v0 + t; v < v1; v += THREADS * DS_UNROLL) {
            if (v != v0 + t) {
#pragma unroll
                for (int u = 0; u < DS_UNROLL; ++u)
                    if (v + u * THREADS < v1) q[u] = __ldg(vec + v + u * THREADS);
            }
#pragma unroll
            for (int u = 0; u < DS_UNROLL; ++u)
                if (v + u * THREADS < v1) {
                    float f[VE];
                    Vec16<T>::unpack(q[u], f);
#pragma unroll
                    for (int i = 0; i < VE; i += 2) unpack2(nothing ? 0ull : slope.pair(f[i], f[i + 1]), f[i], f[i + 1]);
                    __stcs(out + v + u * THREADS, Vec16<T>::pack(f));
                }
        }
        begin = segment == 0 ? 0 : head + v0 * VE;
        end = segment == a.segments - 1 ? a.classes : head + v1 * VE;
        if (segment == 0 && t < head) dx[t] = from_float<T>(nothing ? 0.f : slope.one(to_float(x[t])));
        const int tail = head + nvec * VE + t;
        if (segment == a.segments - 1 && tail < a.classes) dx[tail] = from_float<T>(nothing ? 0.f : slope.one(to_float(x[tail])));
    } else {
        begin = (int)((long long)a.classes * segment / a.segments);
        end = (int)((long long)a.classes * (segment + 1) / a.segments);
        for (int i = begin + t; i < end; i += THREADS) dx[i] = from_float<T>(nothing ? 0.f : slope.one(to_float(x[i])));
    }
    if (nothing) return;
    // The named classes, written again in whole: where several names are one class, each writes the same sum.
    if constexpr (THREADS == 32) __syncwarp(); else __syncthreads();
    for (int j = t; j <= a.k; j += THREADS) {
        const long long i = j < a.k ? at[j] : (gl != 0.f ? target : -1);
        if (i < begin || i >= end) continue;
        float g = i == target ? gl : 0.f;
        for (int l = 0; l < a.k; ++l)
            if (at[l] == i && soft != 0.f) g -= soft * mass[l];
        dx[i] = from_float<T>(slope.one(to_float(x[i])) + g);
    }
}

// A warp a row: short rows, and longer ones where there are enough to fill the SMs.
bool ds_warp_rows(long long rows, long long classes) {
    return classes <= 1024 || (classes <= 4096 && rows >= 8LL * sm_count()) || (classes <= 8192 && rows >= 24LL * sm_count());
}

template <class T, int SECOND> int launch_distill_forward(const DsFwd& a, cudaStream_t s) {
    const auto launch = [&](auto kernel, long long grid, int threads, size_t ring, int parts) {
        const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), ring);
        return st != ADDER_OK ? st : launch_clusters(kernel, (unsigned)grid, threads, ring, parts, s, a);
    };
    if (ds_warp_rows(a.rows, a.classes)) return launch(ds_warp_kernel<T, SECOND>, (a.rows + 3) / 4, 128, LpStream<T, 32>::RING, 1);
    constexpr size_t ring = LpStream<T, DS_TEAM>::RING;
    int parts = 1;      // few rows are split over clusters, as long as there are no more than 4 CTAs an SM
    while (parts < 8 && a.rows * parts * 2 <= sm_count() * 4 && a.classes >= 8192LL * parts) parts *= 2;
    if (parts > 1) return launch(ds_cluster_kernel<T, SECOND>, a.rows * parts, DS_TEAM, ring, parts);
    const long long most = 4LL * sm_count();
    return launch(ds_stream_kernel<T, SECOND>, a.rows < most ? a.rows : most, DS_STREAM, ring, 1);
}

// f(std::integral_constant<int, DsSecond>) by the temperature, and by whether the probabilities at temperature 1 are asked for.
template <class F> int with_second(float temperature, bool asked, F&& f) {
    if (!asked || temperature == 1.f) return f(std::integral_constant<int, ONE>());
    if (temperature == 2.f) return f(std::integral_constant<int, SQUARE>());
    if (temperature == 4.f) return f(std::integral_constant<int, FOURTH>());
    return f(std::integral_constant<int, OWN>());
}

int ds_check(long long rows, long long classes, long long row_stride, int dtype, int k, float temperature) {
    if (rows < 0 || classes <= 0 || k < 1 || (rows > 1 && row_stride < 0) || !(temperature > 0.f) || temperature == INFINITY) return ADDER_ERR_BAD_SHAPE;
    if ((float)(1.4426950408889634 / temperature) == INFINITY) return ADDER_ERR_BAD_SHAPE;      // 0 times it, of the largest logit, would be NaN
    if (classes > 2147483647LL - 1024 || rows > 2147483647LL / 8 || k > DS_MAX_K || dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16) return ADDER_ERR_UNSUPPORTED;
    return ADDER_OK;
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_distillation_forward(const void* logits, int dtype, long long rows, long long classes, long long row_stride, const void* teacher,
                                    int teacher_dtype, const long long* indices, int k, float temperature, const long long* targets,
                                    long long ignore_index, float* divergence, float* log_prob, float* stats, float* mass, void* stream) {
    const int st = ds_check(rows, classes, row_stride, dtype, k, temperature);
    if (st != ADDER_OK) return st;
    if (teacher_dtype < ADDER_TYPE_F32 || teacher_dtype > ADDER_TYPE_F16) return ADDER_ERR_UNSUPPORTED;
    if (rows == 0) return ADDER_OK;
    if (!logits || !teacher || !indices || !divergence || !targets != !log_prob || !stats != !mass) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(logits, dtype == ADDER_TYPE_F32 ? 4 : 2) || !aligned_to(teacher, teacher_dtype == ADDER_TYPE_F32 ? 4 : 2) || !aligned_to(indices, 8) ||
        !aligned_to(targets, 8) || !aligned_to(divergence, 4) || !aligned_to(log_prob, 4) || !aligned_to(stats, 4) || !aligned_to(mass, 4))
        return ADDER_ERR_ALIGNMENT;
    const DsFwd a{logits, rows, row_stride, (int)classes, k, teacher, teacher_dtype, indices, targets, ignore_index, (float)(1.0 / temperature),
                  (float)(1.4426950408889634 / temperature), divergence, log_prob, stats, mass};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return with_second(temperature, targets != nullptr, [&](auto second) { return launch_distill_forward<T, decltype(second)::value>(a, s); });
    });
}

int adder_b200_distillation_backward(const void* logits, int dtype, long long rows, long long classes, long long row_stride,
                                     const long long* indices, int k, float temperature, const long long* targets, long long ignore_index,
                                     const float* stats, const float* mass, const float* grad_divergence, const float* grad_log_prob,
                                     void* grad_logits, void* stream) {
    const int st = ds_check(rows, classes, row_stride, dtype, k, temperature);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!logits || !indices || !stats || !mass || !grad_logits || (grad_log_prob && !targets)) return ADDER_ERR_NULL_POINTER;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!aligned_to(logits, size) || !aligned_to(grad_logits, size) || !aligned_to(indices, 8) || !aligned_to(targets, 8) || !aligned_to(stats, 4) ||
        !aligned_to(mass, 4) || !aligned_to(grad_divergence, 4) || !aligned_to(grad_log_prob, 4))
        return ADDER_ERR_ALIGNMENT;
    const bool warps = ds_warp_rows(rows, classes);
    // A CTA takes two turns, whose loads and stores overlap, or one where there would be too few CTAs.
    const long long turn = (long long)DS_TEAM * DS_UNROLL * (16 / size), ones = (classes + turn - 1) / turn;
    const long long segments = warps ? 1 : rows * ones >= 8LL * sm_count() ? (ones + 1) / 2 : ones;
    const long long grid = warps ? (rows + 3) / 4 : rows * segments;
    if (grid > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    const DsBwd a{logits, rows, row_stride, (int)classes, k, indices, targets, ignore_index, (float)(1.0 / temperature),
                  (float)(1.4426950408889634 / temperature), stats, mass, grad_divergence, grad_log_prob, grad_logits, (int)segments};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return with_second(temperature, grad_log_prob != nullptr, [&](auto second) {
            constexpr int SECOND = decltype(second)::value;
            if (warps) ds_backward_kernel<T, 32, SECOND><<<(unsigned)grid, 128, 0, s>>>(a);
            else ds_backward_kernel<T, DS_TEAM, SECOND><<<(unsigned)grid, DS_TEAM, 0, s>>>(a);
            return launched();
        });
    });
}

}  // extern "C"
