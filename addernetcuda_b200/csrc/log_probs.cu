// Log probabilities of given classes, entropy and the most probable classes of rows of logits, and their gradient.
//
//   forward   M = max x, s = sum e^(x - M);  log p_i = x_i - M - ln s;  H = ln s - sum e^(x - M) (x - M) / s
//             the k largest x with their indices, equal values by index
//   backward  dx_i = -p_i (G + gH (log p_i + H)) + sum over selected j with index i of g_j,  G = sum of all g_j
//             (selected: the target and the k largest)
//
// The forward reads the logits once: every thread keeps a maximum of its own with the two sums relative to it, which are rescaled when
// it rises, and the threads' triples are joined at the end.  The largest k need no second pass over the row either: the k-th largest of
// the threads' maxima is a lower bound of the k-th largest value, so all candidates lie with the at most k threads (and those
// that tie with them) whose maximum reaches it, and only their share of the row is read again.  The backward reads the logits and writes
// the gradient.  Both are bound by memory for large rows; few rows are split over a cluster of CTAs that join through shared memory.
#include "kernels.h"
#include "elements.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace adder {
namespace {

namespace cg = cooperative_groups;

constexpr int LP_MAX_K = 32;
constexpr int LP_TEAM = 256;            // threads of a CTA that has a row, or a part of one, to itself
constexpr int LP_UNROLL = 4;            // vectors that a thread has in flight
constexpr float LP_FLOOR = -200.f;      // 2^-200 is 0 in fp32: stands for exponents of -inf where 0 * -inf would be NaN
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A key orders elements by value, then by index from the lowest: no two are equal.  0 is below all of them.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
    uint32_t u = __float_as_uint(v + 0.f);      // -0 and 0 are one value
    u ^= (uint32_t)((int32_t)u >> 31) | 0x80000000u;
    return ((uint64_t)u << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

__device__ __forceinline__ uint64_t bigger(uint64_t a, uint64_t b) { return a > b ? a : b; }
// Descending order over the lanes of a warp.
__device__ __forceinline__ uint64_t merge_down(uint64_t key, int lane, int width) {
    for (int off = width >> 1; off > 0; off >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, key, off);
        key = ((lane & off) == 0) == (key > other) ? key : other;
    }
    return key;
}
__device__ __forceinline__ uint64_t sort_warp(uint64_t key, int lane) {
#pragma unroll
    for (int width = 2; width <= 32; width <<= 1) {
        // bitonic: every other run of `width` lanes ascends, until the last
        const bool down = (lane & width) == 0 || width == 32;
        for (int off = width >> 1; off > 0; off >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, key, off);
            key = (((lane & off) == 0) == down) == (key > other) ? key : other;
        }
    }
    return key;
}

struct LpFwd {
    const void* x;
    long long rows, stride;
    int classes, k;
    const long long* targets;
    long long ignore;
    float* log_prob;      // may be null, as all of the following
    float* entropy;
    float* stats;         // [rows][2]: M, s
    float* top_log_probs;
    long long* top_indices;
};

// Threads that share a row: a warp, or a CTA (which may be one of a cluster).
template <int THREADS> struct Team {
    static __device__ __forceinline__ void sync() {
        if constexpr (THREADS == 32) __syncwarp(); else __syncthreads();
    }
};

// What a team keeps in shared memory.
template <int THREADS, int LIST> struct LpShared {
    float m[THREADS / 32], s[THREADS / 32], t[THREADS / 32];
    float row[3];                          // M, s, t of the team, then of the row
    uint64_t sorted[THREADS / 32][32];     // sorted maxima of each warp
    uint64_t top[32];                      // the best so far, sorted
    uint64_t list[LIST];                   // candidates
    int winners[THREADS];
    int count, winner_count;
};

// Joins (m, s, t) of two parts: sums relative to the larger maximum.  Equal maxima (both -inf among them) need no factor, and a sum that
// is NaN stays one.
__device__ __forceinline__ void join(float& m, float& s, float& t, float m2, float s2, float t2) {
    const float M = fmaxf(m, m2);
    const float d1 = m == M ? 0.f : fmaxf((m - M) * LOG2E, LP_FLOOR), d2 = m2 == M ? 0.f : fmaxf((m2 - M) * LOG2E, LP_FLOOR);
    const float f1 = exp2_fast(d1), f2 = exp2_fast(d2);
    t = (t + s * d1) * f1 + (t2 + s2 * d2) * f2;
    s = s * f1 + s2 * f2;
    m = M;
}

// The 32 largest of one key a thread, sorted, in the lanes of the team's first warp (others: nothing of use).
template <int THREADS, class Shared> __device__ __forceinline__ uint64_t team_top32(uint64_t key, int t, Shared& sh) {
    const int lane = t & 31, warp = t >> 5;
    key = sort_warp(key, lane);
    if constexpr (THREADS > 32) {
        for (int half = THREADS / 64; half > 0; half >>= 1) {
            if (warp >= half && warp < 2 * half) sh.sorted[warp][lane] = key;
            __syncthreads();
            if (warp < half) key = merge_down(bigger(key, sh.sorted[warp + half][31 - lane]), lane, 32);
        }
    }
    return key;
}

template <class T> __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max_pair<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <> __device__ __forceinline__ uint32_t max_pair<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The largest of a vector's values, NaN if one is: as a word of its type, so that 16-bit values are compared in pairs.
template <class T> __device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    else return max_pair<T>(a, b);
}
template <class T> __device__ __forceinline__ float word_max(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(w);
    } else {
        const float2 p = unpack_pair<T>(w);
        return max_nan(p.x, p.y);
    }
}

// A thread's maximum m with s = sum 2^d and t = sum 2^d d over its values x, d = x log2(e) - ref.  ref is m log2(e) rounded (one fused
// multiply-add a value); what it was rounded by is kept in `res` and comes off at the end.  Beyond |m| = 8192, where the rounding is no longer
// small, d is (x - m) log2(e).
template <bool ENTROPY> struct Running {
    float m = -INFINITY, ref = 0.f, res = 0.f;
    uint64_t s = 0, t = 0;      // pairs of fp32 sums

    __device__ __forceinline__ bool small() const { return fabsf(m) < 8192.f; }
    __device__ __forceinline__ void shift(float d) {
        d = fmaxf(d, LP_FLOOR);
        const float f = exp2_fast(d);
        const uint64_t f2 = pack2(f, f);
        if (ENTROPY) t = fma2(fma2(s, pack2(d, d), t), f2, 0);
        s = fma2(s, f2, 0);
    }
    __device__ __forceinline__ void raise(float top) {
        const float ref_new = top * LOG2E, res_new = fabsf(top) < 8192.f ? fmaf(top, LOG2E, -ref_new) : 0.f;
        shift((m - top) * LOG2E + (res_new - res));
        m = top; ref = ref_new; res = res_new;
    }
    // N values (N even), the largest of which is `top`
    template <int N> __device__ __forceinline__ void take(const float (&f)[N], float top) {
        if (top > m) raise(top);
        if (m == -INFINITY && top == -INFINITY) return;      // nothing so far
        if (small()) {
            const uint64_t scale = pack2(LOG2E, LOG2E), minus = pack2(-ref, -ref);
#pragma unroll
            for (int i = 0; i < N; i += 2) add(fma2(pack2(f[i], f[i + 1]), scale, minus));
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) add(pack2((f[i] - m) * LOG2E, (f[i + 1] - m) * LOG2E));
        }
    }
    __device__ __forceinline__ void add(uint64_t pair) {
        float d0, d1;
        unpack2(pair, d0, d1);
        if (ENTROPY) { d0 = max_nan(d0, LP_FLOOR); d1 = max_nan(d1, LP_FLOOR); }
        const uint64_t e = pack2(exp2_fast(d0), exp2_fast(d1));
        s = add2(s, e);
        if (ENTROPY) t = fma2(e, pack2(d0, d1), t);
    }
    // Sums relative to m itself
    __device__ __forceinline__ void finish(float* sum, float* dot) {
        float a, b;
        unpack2(s, a, b);
        const float all = a + b;
        unpack2(t, a, b);
        const float f = exp2f(-res);
        *sum = all * f;
        *dot = ENTROPY ? ((a + b) - all * res) * f : 0.f;
    }
};

// U vectors of a thread, THREADS apart from the v-th on: their values into the running sums, their maximum into `best`.
template <class T, int THREADS, int U, bool ENTROPY, bool TOP>
__device__ __forceinline__ void take_vectors(const uint4* vec, int v, Running<ENTROPY>& run, float& best, int& best_vec) {
    constexpr int VE = Vec16<T>::N;
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = __ldg(vec + v + u * THREADS);
    uint32_t w[U], all;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        w[u] = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
        all = u == 0 ? w[0] : max_word<T>(all, w[u]);
    }
    const float top = word_max<T>(all);
    if (TOP && top > best) {
        best = top;
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
            if (word_max<T>(w[u]) == top) best_vec = v + u * THREADS;
    }
    float f[U * VE];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float g[VE];
        Vec16<T>::unpack(q[u], g);
#pragma unroll
        for (int i = 0; i < VE; ++i) f[u * VE + i] = g[i];
    }
    run.take(f, top);
}

// grid: rows (times the cluster's size), or rows / 4 with a warp a row
template <class T, int THREADS, bool CLUSTER, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS, THREADS == 32 ? 8 : 1024 / THREADS) lp_forward_kernel(const LpFwd a) {
    constexpr int VE = Vec16<T>::N;
    constexpr int TEAMS = THREADS == 32 ? 4 : 1;
    constexpr int LIST = TOP ? THREADS * VE + 2 * VE : 1;
    __shared__ LpShared<THREADS, LIST> shared[TEAMS];
    const int t = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int team = THREADS == 32 ? threadIdx.x >> 5 : 0;
    LpShared<THREADS, LIST>& sh = shared[team];
    int rank = 0, parts = 1;
    long long row;
    if constexpr (CLUSTER) {
        rank = (int)cg::this_cluster().block_rank();
        parts = (int)cg::this_cluster().num_blocks();
        row = blockIdx.x / parts;
    } else {
        row = (long long)blockIdx.x * TEAMS + team;
        if (row >= a.rows) return;      // whole warps only, and warps of a CTA do not wait for one another
    }
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    // The row's aligned vectors, shared out over the cluster; up to VE - 1 single elements before and behind them are rank 0's.
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int head = min(a.classes, mis == 0 ? 0 : VE - mis);
    const int nvec = (a.classes - head) / VE;
    const int singles = rank == 0 ? a.classes - nvec * VE : 0;
    const int v0 = (int)((long long)nvec * rank / parts), v1 = (int)((long long)nvec * (rank + 1) / parts);
    const uint4* vec = reinterpret_cast<const uint4*>(x + head);
    const auto single_index = [&](int i) { return i < head ? i : i + nvec * VE; };

    Running<ENTROPY> run;
    float best = -INFINITY;
    int best_vec = v0 + t;
    int v = v0 + t;
    for (; v + (LP_UNROLL - 1) * THREADS < v1; v += THREADS * LP_UNROLL) take_vectors<T, THREADS, LP_UNROLL, ENTROPY, TOP>(vec, v, run, best, best_vec);
    for (; v < v1; v += THREADS) take_vectors<T, THREADS, 1, ENTROPY, TOP>(vec, v, run, best, best_vec);
    if (t < singles) {
        const float f[2] = {to_float(x[single_index(t)]), -INFINITY};
        run.take(f, f[0]);
    }
    float m = run.m, s, tt;
    run.finish(&s, &tt);

    // ---- the team's sums
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                    t2 = ENTROPY ? __shfl_xor_sync(0xffffffffu, tt, off) : 0.f;
        join(m, s, tt, m2, s2, t2);
    }
    if constexpr (THREADS > 32) {
        if ((t & 31) == 0) { sh.m[t >> 5] = m; sh.s[t >> 5] = s; sh.t[t >> 5] = tt; }
        __syncthreads();
        if (t < 32) {
            const bool in = t < THREADS / 32;
            m = in ? sh.m[t] : -INFINITY; s = in ? sh.s[t] : 0.f; tt = in ? sh.t[t] : 0.f;
#pragma unroll
            for (int off = THREADS / 64; off > 0; off >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                            t2 = ENTROPY ? __shfl_xor_sync(0xffffffffu, tt, off) : 0.f;
                join(m, s, tt, m2, s2, t2);
            }
        }
    }
    if (t == 0) { sh.row[0] = m; sh.row[1] = s; sh.row[2] = tt; }

    // ---- the team's k largest
    if constexpr (TOP) {
        const bool has = v0 + t < v1;
        const uint32_t lowest = (uint32_t)(head + best_vec * VE);
        // bounds of the thread's largest key, which is in best_vec
        const uint64_t low = has ? key_of(best, lowest + VE - 1) : 0, high = has ? key_of(best, lowest) : 0;
        const uint64_t maxima = team_top32<THREADS>(low, t, sh);
        if (t < 32) sh.top[t] = maxima;
        if (t == 0) { sh.winner_count = 0; sh.count = 0; }
        Team<THREADS>::sync();
        const uint64_t bound = sh.top[a.k - 1];
        Team<THREADS>::sync();
        if (t < 32) sh.top[t] = 0;
        if (has && high >= bound) sh.winners[atomicAdd(&sh.winner_count, 1)] = t;
        Team<THREADS>::sync();
        const int per = (v1 - v0 + THREADS - 1) / THREADS;      // vectors of a thread, the last perhaps not there
        const int items = sh.winner_count * per;
        if (t < singles) {
            const uint32_t i = (uint32_t)single_index(t);
            const uint64_t key = key_of(to_float(x[i]), i);
            if (key >= bound) sh.list[atomicAdd(&sh.count, 1)] = key;
        }
        for (int base = 0; base == 0 || base < items; base += THREADS) {
            const int item = base + t;
            if (item < items) {
                const int v = v0 + sh.winners[item / per] + (item % per) * THREADS;
                if (v < v1) {
                    float g[VE];
                    Vec16<T>::unpack(__ldg(vec + v), g);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const uint64_t key = key_of(g[i], (uint32_t)(head + v * VE + i));
                        if (key >= bound) sh.list[atomicAdd(&sh.count, 1)] = key;
                    }
                }
            }
            Team<THREADS>::sync();
            const int n = sh.count;
            for (int at = 0; at < n; at += THREADS) {
                const uint64_t batch = team_top32<THREADS>(at + t < n ? sh.list[at + t] : 0, t, sh);
                if (t < 32) sh.top[t] = merge_down(bigger(batch, sh.top[31 - t]), t, 32);
                Team<THREADS>::sync();
            }
            if (t == 0) sh.count = 0;
            Team<THREADS>::sync();
        }
    }

    // ---- the row
    if constexpr (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0 && t < 32) {
            for (int r = 1; r < parts; ++r) {
                LpShared<THREADS, LIST>* other = cluster.map_shared_rank(&sh, r);
                if (t == 0) {
                    m = sh.row[0]; s = sh.row[1]; tt = sh.row[2];
                    join(m, s, tt, other->row[0], other->row[1], other->row[2]);
                    sh.row[0] = m; sh.row[1] = s; sh.row[2] = tt;
                }
                if (TOP) {
                    const uint64_t key = merge_down(bigger(sh.top[t], other->top[31 - t]), t, 32);
                    __syncwarp();
                    sh.top[t] = key;
                    __syncwarp();
                }
            }
        }
        cluster.sync();      // no CTA leaves while its shared memory is read
        if (rank != 0) return;
    }
    if (t >= 32) return;
    __syncwarp();
    m = sh.row[0]; s = sh.row[1]; tt = sh.row[2];
    const bool nothing = s == 0.f, broken = s != s;      // all -inf; a NaN or +inf among the logits
    const float ln_s = nothing ? 0.f : logf(s);
    if (t == 0) {
        if (a.stats != nullptr) {
            a.stats[2 * row] = m;
            a.stats[2 * row + 1] = s;
        }
        if (a.log_prob != nullptr) {
            const long long target = a.targets[row];
            float lp = 0.f;
            if (target != a.ignore) {
                if (target < 0 || target >= a.classes || broken) lp = NAN;
                else lp = nothing ? -INFINITY : (to_float(x[target]) - m) - ln_s;
            }
            a.log_prob[row] = lp;
        }
        if (ENTROPY) a.entropy[row] = broken ? NAN : nothing ? 0.f : LN2 * (log2f(s) - tt / s);
    }
    if (TOP && t < a.k) {
        const uint64_t key = sh.top[t];
        a.top_log_probs[row * a.k + t] = broken ? NAN : nothing ? -INFINITY : (key_value(key) - m) - ln_s;
        a.top_indices[row * a.k + t] = broken ? -1 : (long long)key_index(key);
    }
}

struct LpBwd {
    const void* x;
    long long rows, stride;
    int classes, k;
    const long long* targets;
    long long ignore;
    const float* stats;
    const float* entropy;
    const long long* top_indices;
    const float* g_log_prob;      // null: no gradient from there, as the two below
    const float* g_entropy;
    const float* g_top;
    void* dx;
    int segments;                 // parts of a row, each a CTA's (or warp's)
};

// The slope of a row's sum with respect to its logits, without what the selected classes add: -p (G + gH (log p + H)) with
// p = 2^(x log2(e) - ref) scale, so that a value takes one fused multiply-add before its exponential.  What ref is rounded by is in
// `scale` and `shift`; beyond |M| = 8192, where that is no longer small, M is subtracted first.
template <bool ENTROPY> struct Slope {
    float minus, ref, scale, g_ent, shift, sum;      // scale: -G / s, or -1 / s with an entropy
    bool nothing;

    __device__ __forceinline__ void set(float m, float s, float sum_, float g_ent_, float h) {
        nothing = s == 0.f;
        const bool small = fabsf(m) < 8192.f;
        minus = small ? 0.f : m;
        ref = small ? m * LOG2E : 0.f;
        const float res = small ? fmaf(m, LOG2E, -ref) : 0.f;
        sum = sum_; g_ent = g_ent_;
        scale = -exp2f(-res) / s * (ENTROPY ? 1.f : sum);
        shift = ENTROPY ? h - logf(s) - res * LN2 : 0.f;
    }
    // `far`: M is subtracted first
    __device__ __forceinline__ uint64_t pair(float a, float b, bool far) const {
        const uint64_t x = far ? add2(pack2(a, b), pack2(-minus, -minus)) : pack2(a, b);
        float d0, d1;
        unpack2(fma2(x, pack2(LOG2E, LOG2E), pack2(-ref, -ref)), d0, d1);
        if (ENTROPY) { d0 = max_nan(d0, LP_FLOOR); d1 = max_nan(d1, LP_FLOOR); }
        const uint64_t e = fma2(pack2(exp2_fast(d0), exp2_fast(d1)), pack2(scale, scale), 0);
        if (!ENTROPY) return e;
        // d log(2) + H - ln s is log p + H
        const uint64_t lp = fma2(pack2(d0, d1), pack2(LN2, LN2), pack2(shift, shift));
        return fma2(e, fma2(lp, pack2(g_ent, g_ent), pack2(sum, sum)), 0);
    }
    __device__ __forceinline__ float one(float v) const {
        if (nothing) return 0.f;
        float a, b;
        unpack2(pair(v, v, minus != 0.f), a, b);
        return a;
    }
};

// Rows go from the last to the first: the forward call has just read them in the other order, and the last ones are still in L2.
template <class T, int THREADS, bool ENTROPY>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) lp_backward_kernel(const LpBwd a) {
    constexpr int VE = Vec16<T>::N;
    constexpr int TEAMS = THREADS == 32 ? 4 : 1;
    const int t = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    const long long unit = (long long)blockIdx.x * TEAMS + (THREADS == 32 ? threadIdx.x >> 5 : 0);
    const long long line = unit / a.segments;
    const int segment = (int)(unit - line * a.segments);
    if (line >= a.rows) return;
    const long long row = a.rows - 1 - line;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* dx = static_cast<T*>(a.dx) + row * (long long)a.classes;

    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int head = min(a.classes, mis == 0 ? 0 : VE - mis);
    const int nvec = (a.classes - head) / VE;
    const int v0 = (int)((long long)nvec * segment / a.segments), v1 = (int)((long long)nvec * (segment + 1) / a.segments);
    const uint4* vec = reinterpret_cast<const uint4*>(x + head);
    uint4 q[LP_UNROLL];      // in flight while the row's numbers arrive
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u)
        if (same && v0 + t + u * THREADS < v1) q[u] = __ldg(vec + v0 + t + u * THREADS);

    const long long target = a.targets != nullptr ? a.targets[row] : a.ignore;
    float g_target = 0.f;
    if (a.g_log_prob != nullptr && target != a.ignore) g_target = target >= 0 && target < a.classes ? a.g_log_prob[row] : NAN;
    float sum = g_target;
    if (a.g_top != nullptr)
        for (int j = 0; j < a.k; ++j) sum += a.g_top[row * a.k + j];
    Slope<ENTROPY> slope;
    slope.set(a.stats[2 * row], a.stats[2 * row + 1], sum, ENTROPY ? a.g_entropy[row] : 0.f, ENTROPY ? a.entropy[row] : 0.f);

    int begin, end;      // elements of this segment
    if (same) {
        uint4* out = reinterpret_cast<uint4*>(dx + head);
        const auto put = [&](const uint4& in, int v, bool far) {
            float f[VE];
            Vec16<T>::unpack(in, f);
#pragma unroll
            for (int i = 0; i < VE; i += 2) unpack2(slope.pair(f[i], f[i + 1], far), f[i], f[i + 1]);
            __stcs(out + v, Vec16<T>::pack(f));
        };
        for (int v = v0 + t; v < v1; v += THREADS * LP_UNROLL) {
            if (v != v0 + t) {
#pragma unroll
                for (int u = 0; u < LP_UNROLL; ++u)
                    if (v + u * THREADS < v1) q[u] = __ldg(vec + v + u * THREADS);
            }
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u)
                if (v + u * THREADS < v1) {
                    if (slope.nothing) out[v + u * THREADS] = make_uint4(0, 0, 0, 0);
                    else if (slope.minus == 0.f) put(q[u], v + u * THREADS, false);
                    else put(q[u], v + u * THREADS, true);
                }
        }
        begin = segment == 0 ? 0 : head + v0 * VE;
        end = segment == a.segments - 1 ? a.classes : head + v1 * VE;
        if (t < VE && segment == 0 && t < head) dx[t] = from_float<T>(slope.one(to_float(x[t])));
        const int tail = head + nvec * VE + t;
        if (t < VE && segment == a.segments - 1 && tail < a.classes) dx[tail] = from_float<T>(slope.one(to_float(x[tail])));
    } else {
        begin = (int)((long long)a.classes * segment / a.segments);
        end = (int)((long long)a.classes * (segment + 1) / a.segments);
        for (int i = begin + t; i < end; i += THREADS) dx[i] = from_float<T>(slope.one(to_float(x[i])));
    }
    // The selected classes, written again in whole: where two selections name one class, each writes the same sum.
    Team<THREADS>::sync();
    if (slope.nothing) return;
    const int selected = a.g_top != nullptr ? a.k : 0;
    for (int j = t; j <= selected; j += THREADS) {
        const long long i = j < selected ? a.top_indices[row * a.k + j] : (a.g_log_prob != nullptr && target != a.ignore ? target : -1);
        if (i < begin || i >= end) continue;
        float g = i == target ? g_target : 0.f;
        for (int l = 0; l < selected; ++l)
            if (a.top_indices[row * a.k + l] == i) g += a.g_top[row * a.k + l];
        dx[i] = from_float<T>(slope.one(to_float(x[i])) + g);
    }
}

template <class T, int THREADS, bool CLUSTER, bool ENTROPY, bool TOP> int launch_forward(const LpFwd& a, int parts, cudaStream_t s) {
    const auto kernel = lp_forward_kernel<T, THREADS, CLUSTER, ENTROPY, TOP>;
    if constexpr (CLUSTER) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a.rows * parts));
        cfg.blockDim = dim3(THREADS);
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
            (void)cudaGetLastError();
            return ADDER_ERR_CUDA;
        }
        count_launch();
        return ADDER_OK;
    } else {
        const long long grid = THREADS == 32 ? (a.rows + 3) / 4 : a.rows;
        kernel<<<(unsigned)grid, THREADS == 32 ? 128 : THREADS, 0, s>>>(a);
        return launched();
    }
}

template <class T, int THREADS, bool CLUSTER> int choose_forward(const LpFwd& a, int parts, cudaStream_t s) {
    if (a.entropy != nullptr)
        return a.k > 0 ? launch_forward<T, THREADS, CLUSTER, true, true>(a, parts, s) : launch_forward<T, THREADS, CLUSTER, true, false>(a, parts, s);
    return a.k > 0 ? launch_forward<T, THREADS, CLUSTER, false, true>(a, parts, s) : launch_forward<T, THREADS, CLUSTER, false, false>(a, parts, s);
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_log_probs_forward(const void* logits, int dtype, long long rows, long long classes, long long row_stride,
                                 const long long* targets, long long ignore_index, int top_k, float* log_prob, float* entropy,
                                 float* stats, float* top_log_probs, long long* top_indices, void* stream) {
    if (rows < 0 || classes <= 0 || top_k < 0 || top_k > classes || (rows > 1 && row_stride < 0)) return ADDER_ERR_BAD_SHAPE;
    if (classes > 2147483647LL - 1024 || rows > 2147483647LL || top_k > LP_MAX_K) return ADDER_ERR_UNSUPPORTED;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16) return ADDER_ERR_UNSUPPORTED;
    if (rows == 0) return ADDER_OK;
    if (!logits || (log_prob && !targets) || (top_k > 0 && (!top_log_probs || !top_indices))) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(logits, dtype == ADDER_TYPE_F32 ? 4 : 2)) return ADDER_ERR_ALIGNMENT;
    const LpFwd a{logits, rows, row_stride, (int)classes, top_k, targets, ignore_index, log_prob, entropy, stats, top_log_probs, top_indices};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        if (classes <= 1024) return choose_forward<T, 32, false>(a, 1, s);
        // Few rows leave SMs idle: a row is then split over a cluster of up to 8 CTAs of at least 4096 elements.
        int parts = 1;
        while (parts < 8 && rows * parts * 2 <= sm_count() * 2 && classes >= 8192LL * parts) parts *= 2;
        if (parts > 1) return choose_forward<T, LP_TEAM, true>(a, parts, s);
        return choose_forward<T, LP_TEAM, false>(a, 1, s);
    });
}

int adder_b200_log_probs_backward(const void* logits, int dtype, long long rows, long long classes, long long row_stride,
                                  const long long* targets, long long ignore_index, int top_k, const long long* top_indices,
                                  const float* stats, const float* entropy, const float* grad_log_prob, const float* grad_entropy,
                                  const float* grad_top, void* grad_logits, void* stream) {
    if (rows < 0 || classes <= 0 || top_k < 0 || top_k > classes || (rows > 1 && row_stride < 0)) return ADDER_ERR_BAD_SHAPE;
    if (classes > 2147483647LL - 1024 || rows > 2147483647LL || top_k > LP_MAX_K) return ADDER_ERR_UNSUPPORTED;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16) return ADDER_ERR_UNSUPPORTED;
    if (rows == 0) return ADDER_OK;
    if (!logits || !stats || !grad_logits || (grad_log_prob && !targets) || (grad_entropy && !entropy) ||
        (grad_top && (top_k == 0 || !top_indices)))
        return ADDER_ERR_NULL_POINTER;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!aligned_to(logits, size) || !aligned_to(grad_logits, size)) return ADDER_ERR_ALIGNMENT;
    const long long tile = 256LL * LP_UNROLL * (16 / size);      // elements that a CTA takes at once
    const bool warps = classes <= 1024;
    const long long segments = warps ? 1 : (classes + tile - 1) / tile;
    const long long grid = warps ? (rows + 3) / 4 : rows * segments;
    if (grid > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    const LpBwd a{logits, rows, row_stride, (int)classes, top_k, targets, ignore_index, stats, entropy, top_indices,
                  grad_log_prob, grad_entropy, grad_top, grad_logits, (int)segments};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        if (warps) {
            if (grad_entropy) lp_backward_kernel<T, 32, true><<<(unsigned)grid, 128, 0, s>>>(a);
            else lp_backward_kernel<T, 32, false><<<(unsigned)grid, 128, 0, s>>>(a);
        } else {
            if (grad_entropy) lp_backward_kernel<T, 256, true><<<(unsigned)grid, 256, 0, s>>>(a);
            else lp_backward_kernel<T, 256, false><<<(unsigned)grid, 256, 0, s>>>(a);
        }
        return launched();
    });
}

}  // extern "C"
