// Log probabilities of given classes, entropy and the most probable classes of rows of logits, and their gradient.
//
//   forward   M = max x, s = sum e^(x - M);  log p_i = x_i - M - ln s;  H = ln s - sum e^(x - M) (x - M) / s
//             the k largest x with their indices, equal values by index
//   backward  dx_i = -p_i (G + gH (log p_i + H)) + sum over selected j with index i of g_j,  G = sum of all g_j
//             (selected: the target and the k largest)
//
// The forward reads the logits once: every thread keeps a maximum of its own with the two sums relative to it, which are rescaled when
// it rises, and the threads' triples are joined at the end, by a warp that does nothing else while the others stream the next row.  The
// largest k need no second pass over the row either: the k-th largest of some of the threads' maxima is a lower bound of the k-th largest
// value, so all candidates lie with the few threads whose maximum reaches it, and only their best group of vectors is read again.  The
// backward reads the logits again and writes the gradient.
//
// What bounds them: memory, at 99 % of a copy's rate for the gradient (2048x128000 bf16: 161 us for 1.05 GB) and for the forward of fp32
// logits (4096x32000: 81 us); the forward of 16-bit logits takes some 8 instructions a value and reaches 90 % (2048x128000
// with entropy 89 us), and 81 % with 50257 classes (4096 rows 77 us; 91 us with the 5 largest, 107 with 20, 126 with 32, which one warp a CTA
// finds while eight stream).  A few rows are split over a cluster of CTAs that join through shared memory (4x32000: 6 us, 10 us with the 20
// largest).  Rows by warps wait for loads and joins: 16384x1000 fp32 18.6 us (54 %), 16384x4000 bf16 with entropy 38 us (53 %), 16384x1000
// bf16 20.6 us (24 %) and with the 5 largest 31.9 (16 %): a warp looks for them alone, after its row.
// The gradient goes by vectors where a row of logits and its row of dx lie alike modulo 16 bytes.  Elsewhere (most rows of a padded buffer
// whose row stride is not the number of classes) it goes element by element: 2048x50257 in rows of 50304 288 us bf16 and 260 fp32, where
// dense rows take 74 and 126.
#include "kernels.h"
#include "elements.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace adder {
namespace {

namespace cg = cooperative_groups;

constexpr int LP_MAX_K = 32;
constexpr int LP_TEAM = 256;            // threads that stream one row; a CTA has one warp more, which finishes rows
constexpr int LP_UNROLL = 4;            // backward: vectors that a thread has in flight
constexpr int LP_GROUP = 4, LP_STAGES = 2;      // forward: vectors of a thread that are taken together, groups of them on their way or in use
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

// Shared memory of the warp that finishes a row.
template <class T, int STREAM, bool TOP> struct LpFinish {
    static constexpr int VECTORS = STREAM == 32 ? 1 : 4;               // of a lane, that are looked at together
    static constexpr int LIST = 96, HOT = VECTORS * 32;
    uint64_t list[TOP ? LIST : 1];         // candidates
    uint64_t sorted[TOP ? 32 : 1];
    uint4 hot[TOP ? HOT : 1];              // vectors that hold some
    int hot_at[TOP ? HOT : 1];
    int first[TOP ? STREAM : 1];           // vectors where the share of a thread begins that may hold some
    uint64_t bound;
    int count;
};
// A thread's largest value and the vector that it is in, and the largest of the groups of vectors that it is not in.
struct Best {
    float value, second;
    int vec;
};
// What the streaming threads hand over: joining it is left to the warp that finishes the row.
struct LpHand {
    float m[LP_TEAM], s[LP_TEAM], t[LP_TEAM];
    Best best[LP_TEAM];
};
// What the CTAs of a cluster leave in the shared memory of the first.
struct LpParts {
    float m[8], s[8], t[8];
    uint64_t top[8][32];
};

// Named barriers between the streaming warps and the finishing one; 0 is __syncthreads.
enum { LP_EMPTY = 1, LP_FULL = 3 };      // two of each
template <int ID> __device__ __forceinline__ void bar_sync(int buffer) {
    if (buffer == 0) asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(LP_TEAM + 32) : "memory");
    else asm volatile("bar.sync %0, %1;" ::"n"(ID + 1), "n"(LP_TEAM + 32) : "memory");
}
template <int ID> __device__ __forceinline__ void bar_arrive(int buffer) {
    if (buffer == 0) asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(LP_TEAM + 32) : "memory");
    else asm volatile("bar.arrive %0, %1;" ::"n"(ID + 1), "n"(LP_TEAM + 32) : "memory");
}

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
    // With an entropy values below this count as this: their exponential is 0 either way, and 0 * -inf would be NaN.  |m| / 64 covers
    // its rounding to 16 bits.
    __device__ __forceinline__ float floor_value() const { return m - 150.f - fabsf(m) * 0.015625f; }

    __device__ __forceinline__ bool small() const { return fabsf(m) < 8192.f; }
    __device__ __forceinline__ void shift(float d) {
        d = fmaxf(d, LP_FLOOR);
        const float f = exp2_fast(d);
        const uint64_t f2 = pack2(f, f);
        if (ENTROPY) t = mul2(fma2(s, pack2(d, d), t), f2);
        s = mul2(s, f2);
    }
    __device__ __forceinline__ void raise(float top) {
        const float ref_new = top * LOG2E, res_new = fabsf(top) < 8192.f ? fmaf(top, LOG2E, -ref_new) : 0.f;
        shift((m - top) * LOG2E + (res_new - res));
        m = top; ref = ref_new; res = res_new;
    }
    // N pairs of values, pair(i, floored) each, the largest of which is `top` and not above m
    template <int N, class Pair> __device__ __forceinline__ void take(Pair&& pair, float top) {
        if (m == -INFINITY && top == -INFINITY) return;      // nothing so far
        if (small()) {
            const uint64_t scale = pack2(LOG2E, LOG2E), minus = pack2(-ref, -ref);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 f = pair(i, ENTROPY);
                add(fma2(pack2(f.x, f.y), scale, minus));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 f = pair(i, false);
                float d0 = (f.x - m) * LOG2E, d1 = (f.y - m) * LOG2E;
                if (ENTROPY) { d0 = max_nan(d0, LP_FLOOR); d1 = max_nan(d1, LP_FLOOR); }
                add(pack2(d0, d1));
            }
        }
    }
    __device__ __forceinline__ void add(uint64_t pair) {
        float d0, d1;
        unpack2(pair, d0, d1);
        const uint64_t e = pack2(exp2_fast(d0), exp2_fast(d1));
        s = add2(s, e);
        if (ENTROPY) t = fma2(e, pair, t);
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

// A row as a team sees it: aligned vectors v0 to v1 - 1 (shared out over the cluster), and up to VE - 1 single elements before and
// behind all vectors, which are rank 0's.
template <class T> struct LpRow {
    static constexpr int VE = Vec16<T>::N;
    const T* x;
    const uint4* vec;
    int head, nvec, singles, v0, v1;

    __device__ __forceinline__ void set(const LpFwd& a, long long row, int rank, int parts) {
        x = static_cast<const T*>(a.x) + row * a.stride;
        const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        head = min(a.classes, mis == 0 ? 0 : VE - mis);
        nvec = (a.classes - head) / VE;
        singles = rank == 0 ? a.classes - nvec * VE : 0;
        v0 = parts == 1 ? 0 : (int)((long long)nvec * rank / parts);
        v1 = parts == 1 ? nvec : (int)((long long)nvec * (rank + 1) / parts);
        vec = reinterpret_cast<const uint4*>(x + head);
    }
    // At least one, so that a row without vectors takes its turn.
    __device__ __forceinline__ int groups(int threads) const { return max(1, (v1 - v0 + LP_GROUP * threads - 1) / (LP_GROUP * threads)); }
    __device__ __forceinline__ int single(int i) const { return i < head ? i : i + nvec * VE; }
};

// A group's values into the running sums, its maximum into `best`.
template <class T, int THREADS, int U, bool ENTROPY, bool TOP>
__device__ __forceinline__ void take_group(const uint4 (&q)[U], int v, Running<ENTROPY>& run, Best& best) {
    constexpr int VE = Vec16<T>::N;
    uint32_t w[U], all;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        w[u] = max_word<T>(max_word<T>(q[u].x, q[u].y), max_word<T>(q[u].z, q[u].w));
        all = u == 0 ? w[0] : max_word<T>(all, w[u]);
    }
    const float top = word_max<T>(all);
    if (TOP) best.second = fmaxf(best.second, fminf(best.value, top));
    if (TOP && top > best.value) {
        best.value = top;
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
            if (word_max<T>(w[u]) == top) best.vec = v + u * THREADS;
    }
    if (top > run.m) run.raise(top);
    const float low = run.floor_value();
    uint32_t low_word = __float_as_uint(low);
    if constexpr (sizeof(T) == 2) low_word = pack_pair<T>(low, low);
    run.template take<U * VE / 2>([&](int i, bool floored) {
        const int u = i / (VE / 2), j = i % (VE / 2);
        if constexpr (sizeof(T) == 4) {
            float2 f = j == 0 ? make_float2(__uint_as_float(q[u].x), __uint_as_float(q[u].y)) : make_float2(__uint_as_float(q[u].z), __uint_as_float(q[u].w));
            if (floored) { f.x = max_nan(f.x, low); f.y = max_nan(f.y, low); }
            return f;
        } else {
            const uint32_t word = j == 0 ? q[u].x : j == 1 ? q[u].y : j == 2 ? q[u].z : q[u].w;
            return unpack_pair<T>(floored ? max_pair<T>(word, low_word) : word);
        }
    }, top);
}

// Sums of a warp's lanes, in every lane.
template <bool ENTROPY> __device__ __forceinline__ void join_lanes(float& m, float& s, float& t, int lanes) {
    for (int off = lanes >> 1; off > 0; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                    t2 = ENTROPY ? __shfl_xor_sync(0xffffffffu, t, off) : 0.f;
        join(m, s, t, m2, s2, t2);
    }
}

__device__ __forceinline__ void copy16(uint32_t to, const uint4* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 read16(uint32_t from) {
    uint4 q;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(from) : "memory");
    return q;
}

// The vectors of a team's rows on their way through shared memory.  Every thread copies what it will read itself, so no thread waits
// for another, and the copies of the next rows go on while a row is finished.
template <class T, int THREADS> struct LpStream {
    static constexpr int CTA = THREADS == 32 ? 128 : THREADS;      // threads that stream
    static constexpr uint32_t SLOT = CTA * 16, STAGE = LP_GROUP * SLOT, RING = LP_STAGES * STAGE;      // bytes
    uint32_t first, at;      // this thread's first slot, and the next to be filled
    const uint4* src;        // of the next group
    int left;                // vectors of the row from there on, in steps of one, of which every THREADS-th is this thread's
    int groups;              // of the row
    long long row, step;

    __device__ __forceinline__ void set_row(const LpFwd& a, int t, int rank, int parts) {
        LpRow<T> r;
        r.set(a, row, rank, parts);
        src = r.vec + r.v0 + t;
        left = r.v1 - r.v0 - t;
        groups = r.groups(THREADS);
    }
    __device__ __forceinline__ void issue(const LpFwd& a, int t, int rank, int parts) {
        if (groups > 0) {
            if (left > (LP_GROUP - 1) * THREADS) {
#pragma unroll
                for (int u = 0; u < LP_GROUP; ++u) copy16(at + u * SLOT, src + u * THREADS);
            } else {
#pragma unroll
                for (int u = 0; u < LP_GROUP - 1; ++u)
                    if (u * THREADS < left) copy16(at + u * SLOT, src + u * THREADS);
            }
            src += LP_GROUP * THREADS;
            left -= LP_GROUP * THREADS;
            if (--groups == 0) {
                row += step;
                if (row < a.rows) set_row(a, t, rank, parts);
            }
        }
        cp_async_commit();
        at = at == first + RING - STAGE ? first : at + STAGE;
    }
};

// The k-th largest of the lanes' keys, 0 where fewer than k lanes have one.  Values first: one round takes all lanes of equal value.
__device__ __forceinline__ uint64_t kth_largest(uint64_t key, int k) {
    uint32_t value = (uint32_t)(key >> 32);
    for (int found = 0;;) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, value);
        if (top == 0) return 0;
        const int n = __popc(__ballot_sync(0xffffffffu, value == top));
        if (found + n < k) {
            found += n;
            if (value == top) value = 0;
            continue;
        }
        uint32_t low = value == top ? (uint32_t)key : 0, last = 0;
        for (; found < k; ++found) {
            last = __reduce_max_sync(0xffffffffu, low);
            if (low == last) low = 0;
        }
        return ((uint64_t)top << 32) | last;
    }
}

// The sums of a row (or of its cluster rank's part) in every lane of one warp, the single elements with them.
template <class T, bool ENTROPY> __device__ __forceinline__ void finish_sums(const LpRow<T>& r, float one, int lane, float& m, float& s, float& t) {
    if (r.singles > 0) {
        Running<ENTROPY> run;
        if (lane < r.singles) {
            if (one > run.m) run.raise(one);
            const float below = run.floor_value();
            run.template take<1>([&](int, bool floored) { return floored ? make_float2(max_nan(one, below), below) : make_float2(one, -INFINITY); }, one);
        }
        float s2, t2;
        run.finish(&s2, &t2);
        join(m, s, t, run.m, s2, t2);
    }
    join_lanes<ENTROPY>(m, s, t, 32);
}

// A bound of a thread's largest key from below (above, with `up`): its best value is somewhere in its vector.
template <class T> __device__ __forceinline__ uint64_t bound_of(const LpRow<T>& r, const Best& f, int thread, bool up) {
    return r.v0 + thread < r.v1 ? key_of(f.value, (uint32_t)(r.head + f.vec * Vec16<T>::N + (up ? 0 : Vec16<T>::N - 1))) : 0;
}

// A key that at least k elements reach, by one warp: the k-th largest best of 32 disjoint sets of threads, one a lane, or, for more than 8, of
// 64 (by sorting, and with some 1.3 k candidates where 32 sets give up to 4 k).  best(i): of thread 32 i + lane.
template <class T, int STREAM, class GetBest> __device__ __forceinline__ uint64_t find_bound(const LpRow<T>& r, int k, int lane, GetBest&& best) {
    constexpr int N = STREAM / 32;
    uint64_t low[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) low[i < (N + 1) / 2 ? 0 : 1] = bigger(low[i < (N + 1) / 2 ? 0 : 1], bound_of(r, best(i), 32 * i + lane, false));
    if (N == 1) return kth_largest(low[0], k);
    if (k <= 8) return kth_largest(bigger(low[0], low[1]), k);
    const uint64_t a = sort_warp(low[0], lane), b = sort_warp(low[1], lane);
    return __shfl_sync(0xffffffffu, merge_down(bigger(a, __shfl_sync(0xffffffffu, b, 31 - lane)), lane, 32), k - 1);
}

// Candidates of one warp, which keeps their number n in every lane.
template <class Finish> struct Candidates {
    Finish& sh;
    int lane, n = 0;
    bool merged = false;
    uint64_t top = 0;      // where there were many: the 32 largest of those taken off the list, sorted

    __device__ __forceinline__ void offer(bool in, uint64_t key) {
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (who == 0) return;
        if (in) sh.list[n + __popc(who & ((1u << lane) - 1))] = key;
        n += __popc(who);
        if (n > Finish::LIST - 32) merge();
    }
    __device__ __forceinline__ void merge() {
        __syncwarp();
        for (int at = 0; at < n; at += 32) {
            const uint64_t batch = sort_warp(at + lane < n ? sh.list[at + lane] : 0, lane);
            const uint64_t other = __shfl_sync(0xffffffffu, top, 31 - lane);
            top = merged ? merge_down(bigger(batch, other), lane, 32) : batch;
            merged = true;
        }
        n = 0;
        __syncwarp();
    }
    // The largest, sorted, one a lane.  Up to 64 candidates each count those above them.
    __device__ __forceinline__ uint64_t finish() {
        if (merged) {
            merge();
            return top;
        }
        __syncwarp();
        sh.sorted[lane] = 0;
        const uint64_t key0 = lane < n ? sh.list[lane] : 0, key1 = lane + 32 < n ? sh.list[lane + 32] : 0;
        int above0 = 0, above1 = 0;
        if (n <= 32) {
            for (int i = 0; i < n; ++i) above0 += sh.list[i] > key0;
        } else {
            for (int i = 0; i < n; ++i) {
                const uint64_t other = sh.list[i];
                above0 += other > key0;
                above1 += other > key1;
            }
        }
        __syncwarp();
        if (lane < n && above0 < 32) sh.sorted[above0] = key0;
        if (lane + 32 < n && above1 < 32) sh.sorted[above1] = key1;
        __syncwarp();
        return sh.sorted[lane];
    }
};

// The k largest of a row, sorted, one a lane of one warp (at least k of the 32).  All candidates lie with the threads whose best reaches the bound:
// in the group of vectors that holds it, and elsewhere in their share only where their second group reaches it, too.  `fetch(v)` reads a
// vector again.
template <class T, int STREAM, class GetBest, class Fetch>
__device__ __forceinline__ uint64_t find_top(const LpRow<T>& r, uint64_t bound, float one, int lane, LpFinish<T, STREAM, true>& sh, GetBest&& best, Fetch&& fetch) {
    using Finish = LpFinish<T, STREAM, true>;
    constexpr int VE = Vec16<T>::N;
    Candidates<Finish> found{sh, lane};
    int one_group = 0, whole = 0;      // threads of which a group of vectors, or all, are looked at
    __syncwarp();
#pragma unroll
    for (int i = 0; i < STREAM / 32; ++i) {
        const Best f = best(i);
        const int thread = 32 * i + lane;
        const uint64_t high = bound_of(r, f, thread, true);
        const bool in = high != 0 && high >= bound, all = in && key_of(f.second, 0) >= bound;
        const unsigned some = __ballot_sync(0xffffffffu, in && !all), every = __ballot_sync(0xffffffffu, all), before = (1u << lane) - 1;
        const int group = (f.vec - r.v0 - thread) / (LP_GROUP * STREAM);
        if (in && !all) sh.first[one_group + __popc(some & before)] = r.v0 + thread + group * LP_GROUP * STREAM;
        if (all) sh.first[STREAM - 1 - whole - __popc(every & before)] = r.v0 + thread;
        one_group += __popc(some);
        whole += __popc(every);
    }
    __syncwarp();
    if (r.singles > 0) {
        const uint64_t key = lane < r.singles ? key_of(one, (uint32_t)r.single(lane)) : 0;
        found.offer(key != 0 && key >= bound, key);
    }
    const int per = (r.v1 - r.v0 + STREAM - 1) / STREAM;      // vectors of a thread, the last perhaps not there
    const int items = one_group * LP_GROUP + whole * per;
    for (int base = 0; base < items; base += Finish::HOT) {
        uint4 p[Finish::VECTORS];
        int at[Finish::VECTORS];
#pragma unroll
        for (int u = 0; u < Finish::VECTORS; ++u) {
            int item = base + 32 * u + lane;
            at[u] = r.v1;
            if (item < one_group * LP_GROUP) {
                at[u] = sh.first[item / LP_GROUP] + item % LP_GROUP * STREAM;
            } else if (item < items) {
                item -= one_group * LP_GROUP;
                const int w = item / per;
                at[u] = sh.first[STREAM - 1 - w] + (item - w * per) * STREAM;
            }
            if (at[u] < r.v1) p[u] = fetch(at[u]);
        }
        int hot = 0;      // vectors that hold a candidate; the elements of those are then looked at one a lane
#pragma unroll
        for (int u = 0; u < Finish::VECTORS; ++u) {
            bool in = false;
            if (at[u] < r.v1)
                in = key_of(word_max<T>(max_word<T>(max_word<T>(p[u].x, p[u].y), max_word<T>(p[u].z, p[u].w))), 0) >= bound;
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (in) {
                const int slot = hot + __popc(who & ((1u << lane) - 1));
                sh.hot[slot] = p[u];
                sh.hot_at[slot] = r.head + at[u] * VE;
            }
            hot += __popc(who);
        }
        __syncwarp();
        for (int e = 0; e < hot * VE; e += 32) {
            const int i = (e + lane) / VE, j = (e + lane) % VE;
            uint64_t key = 0;
            if (i < hot) key = key_of(to_float(reinterpret_cast<const T*>(&sh.hot[i])[j]), (uint32_t)(sh.hot_at[i] + j));
            found.offer(key != 0 && key >= bound, key);
        }
        __syncwarp();
    }
    return found.finish();
}

// The outputs of a row, by one warp whose lanes all have its sums.
template <bool ENTROPY, bool TOP>
__device__ __forceinline__ void write_row(const LpFwd& a, long long row, int lane, float m, float s, float t, uint64_t top, long long target, float at_target) {
    const bool nothing = s == 0.f, broken = s != s;      // all -inf; a NaN or +inf among the logits
    const float ln_s = nothing ? 0.f : logf(s);
    if (lane == 0) {
        if (a.stats != nullptr) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(m, s);
        if (a.log_prob != nullptr) {
            float lp = 0.f;
            if (target != a.ignore) {
                if (target < 0 || target >= a.classes || broken) lp = NAN;
                else lp = nothing ? -INFINITY : (at_target - m) - ln_s;
            }
            a.log_prob[row] = lp;
        }
        if (ENTROPY) a.entropy[row] = broken ? NAN : nothing ? 0.f : LN2 * (log2f(s) - t / s);
    }
    if (TOP && lane < a.k) {
        a.top_log_probs[row * a.k + lane] = broken ? NAN : nothing ? -INFINITY : (key_value(top) - m) - ln_s;
        a.top_indices[row * a.k + lane] = broken ? -1 : (long long)key_index(top);
    }
}

// THREADS threads stream every grid-th row (or, in a cluster, a part of one row).  A warp that has a row to itself finishes it, too; with
// LP_TEAM threads another warp of the CTA does, while they are in the next row.
template <class T, int THREADS, bool CLUSTER, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : LP_TEAM + 32, THREADS == 32 ? 8 : 4) lp_forward_kernel(const LpFwd a) {
    constexpr int TEAMS = THREADS == 32 ? 4 : 1;
    extern __shared__ uint4 ring[];         // [LP_STAGES][LP_GROUP][threads]
    __shared__ LpFinish<T, THREADS, TOP> finishing[TEAMS];
    __shared__ LpHand hand[THREADS == 32 ? 1 : 2];
    __shared__ LpParts joined[1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = THREADS == 32 ? lane : threadIdx.x;
    int rank = 0, parts = 1;
    long long row, step;
    if constexpr (CLUSTER) {
        rank = (int)cg::this_cluster().block_rank();
        parts = (int)cg::this_cluster().num_blocks();
        row = blockIdx.x / parts;
        step = a.rows;      // a cluster has one row
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");      // waited for before the first word crosses over
    } else {
        row = (long long)blockIdx.x * TEAMS + (THREADS == 32 ? warp : 0);
        step = (long long)gridDim.x * TEAMS;
    }
    if (row >= a.rows) return;      // whole warps only, and warps of a CTA do not wait for one another
    LpFinish<T, THREADS, TOP>& sh = finishing[THREADS == 32 ? warp : 0];
    const bool finisher = warp == LP_TEAM / 32;

    if constexpr (THREADS > 32) if (finisher) {
        __syncwarp();
        if (!CLUSTER) {      // where there is one row, nobody waits for these
            bar_arrive<LP_EMPTY>(0);
            if (row + step < a.rows) bar_arrive<LP_EMPTY>(1);
        }
        int buffer = 0;
        long long target_next = a.log_prob != nullptr ? a.targets[row] : 0;
        for (; row < a.rows; row += step) {
            LpRow<T> r;
            r.set(a, row, rank, parts);
            const long long target = target_next;
            const float at_target = a.log_prob != nullptr && target >= 0 && target < a.classes ? to_float(r.x[target]) : 0.f;
            if (a.log_prob != nullptr && row + step < a.rows) target_next = a.targets[row + step];
            const float one = lane < r.singles ? to_float(r.x[r.single(lane)]) : -INFINITY;
            __syncwarp();
            bar_sync<LP_FULL>(buffer);
            const LpHand& in = hand[buffer];
            float m = in.m[lane], s = in.s[lane], tt = ENTROPY ? in.t[lane] : 0.f;
#pragma unroll
            for (int i = 1; i < LP_TEAM / 32; ++i) join(m, s, tt, in.m[32 * i + lane], in.s[32 * i + lane], ENTROPY ? in.t[32 * i + lane] : 0.f);
            finish_sums<T, ENTROPY>(r, one, lane, m, s, tt);
            uint64_t top = 0;
            if constexpr (TOP) {
                const auto best = [&](int i) { return in.best[32 * i + lane]; };
                const auto fetch = [&](int v) { return __ldg(r.vec + v); };
                const uint64_t bound = find_bound<T, THREADS>(r, a.k, lane, best);
                if constexpr (CLUSTER) {      // few rows: the streaming threads have nothing else to do than to look through their own vectors
                    if (lane == 0) { sh.bound = bound; sh.count = 0; }
                    __syncwarp();
                    bar_sync<LP_EMPTY>(0);
                    bar_sync<LP_EMPTY>(1);
                    Candidates<LpFinish<T, THREADS, TOP>> found{sh, lane, sh.count};
                    if (found.n <= LpFinish<T, THREADS, TOP>::LIST - 32) {
                        if (r.singles > 0) {
                            const uint64_t key = lane < r.singles ? key_of(one, (uint32_t)r.single(lane)) : 0;
                            found.offer(key != 0 && key >= bound, key);
                        }
                        top = found.finish();
                    } else {
                        top = find_top<T, THREADS>(r, bound, one, lane, sh, best, fetch);
                    }
                } else {
                    top = find_top<T, THREADS>(r, bound, one, lane, sh, best, fetch);
                }
            }
            __syncwarp();
            if (row + 2 * step < a.rows) bar_arrive<LP_EMPTY>(buffer);
            buffer ^= 1;
            if constexpr (CLUSTER) {      // every rank hands its part to rank 0
                cg::cluster_group cluster = cg::this_cluster();
                asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
                LpParts* to = cluster.map_shared_rank(&joined[0], 0);
                if (lane == 0) { to->m[rank] = m; to->s[rank] = s; to->t[rank] = tt; }
                if (TOP) to->top[rank][lane] = top;
                cluster.sync();
                if (rank != 0) return;
                const bool there = lane < parts;
                m = there ? joined[0].m[lane] : -INFINITY; s = there ? joined[0].s[lane] : 0.f; tt = there ? joined[0].t[lane] : 0.f;
                join_lanes<ENTROPY>(m, s, tt, 32);
                if constexpr (TOP) {      // by halves: the merges of a round do not depend on one another
                    uint64_t part[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) part[i] = i < parts ? joined[0].top[i][lane] : 0;
#pragma unroll
                    for (int half = 4; half > 0; half >>= 1)
#pragma unroll
                        for (int i = 0; i < half; ++i)
                            part[i] = merge_down(bigger(part[i], __shfl_sync(0xffffffffu, part[i + half], 31 - lane)), lane, 32);
                    top = part[0];
                }
            }
            write_row<ENTROPY, TOP>(a, row, lane, m, s, tt, top, target, at_target);
        }
        return;
    }

    using Stream = LpStream<T, THREADS>;
    Stream stream;
    stream.first = stream.at = smem_u32(ring) + threadIdx.x * 16;
    stream.row = row; stream.step = step;
    stream.set_row(a, t, rank, parts);
#pragma unroll
    for (int i = 0; i < LP_STAGES - 1; ++i) stream.issue(a, t, rank, parts);
    uint32_t from = stream.first;
    int buffer = 0;
    long long target_next = THREADS == 32 && a.log_prob != nullptr ? a.targets[row] : 0;
    for (; row < a.rows; row += step) {
        LpRow<T> r;
        r.set(a, row, rank, parts);
        // what is needed once the row is through
        const long long target = target_next;
        float at_target = 0.f, one = -INFINITY;
        if constexpr (THREADS == 32) {
            if (a.log_prob != nullptr && target >= 0 && target < a.classes) at_target = to_float(r.x[target]);
            if (a.log_prob != nullptr && row + step < a.rows) target_next = a.targets[row + step];
            if (lane < r.singles) one = to_float(r.x[r.single(lane)]);
        }
        Running<ENTROPY> run;
        int v = r.v0 + t;
        Best best{-INFINITY, -INFINITY, v};
        for (int g = r.groups(THREADS); g > 0; --g) {
            stream.issue(a, t, rank, parts);
            cp_async_wait<LP_STAGES - 1>();
            if (v + (LP_GROUP - 1) * THREADS < r.v1) {
                uint4 q[LP_GROUP];
#pragma unroll
                for (int u = 0; u < LP_GROUP; ++u) q[u] = read16(from + u * Stream::SLOT);
                take_group<T, THREADS, LP_GROUP, ENTROPY, TOP>(q, v, run, best);
            } else {
#pragma unroll 1
                for (int u = 0; u < LP_GROUP - 1 && v + u * THREADS < r.v1; ++u) {
                    const uint4 q[1] = {read16(from + u * Stream::SLOT)};
                    take_group<T, THREADS, 1, ENTROPY, TOP>(q, v + u * THREADS, run, best);
                }
            }
            from = from == stream.first + Stream::RING - Stream::STAGE ? stream.first : from + Stream::STAGE;
            v += LP_GROUP * THREADS;
        }
        float m = run.m, s, tt;
        run.finish(&s, &tt);
        if constexpr (THREADS == 32) {
            uint64_t top = 0;
            finish_sums<T, ENTROPY>(r, one, lane, m, s, tt);
            if constexpr (TOP) {
                const auto mine = [&](int) { return best; };
                top = find_top<T, 32>(r, find_bound<T, 32>(r, a.k, lane, mine), one, lane, sh, mine, [&](int v) { return __ldg(r.vec + v); });
            }
            write_row<ENTROPY, TOP>(a, row, lane, m, s, tt, top, target, at_target);
        } else {
            __syncwarp();
            if (!CLUSTER) bar_sync<LP_EMPTY>(buffer);
            LpHand& out = hand[buffer];
            out.m[t] = m; out.s[t] = s;
            if (ENTROPY) out.t[t] = tt;
            if (TOP) out.best[t] = best;
            __syncwarp();
            bar_arrive<LP_FULL>(buffer);
            buffer ^= 1;
            if constexpr (CLUSTER && TOP) {      // candidates of this thread, as long as the list has room for all
                bar_sync<LP_EMPTY>(0);
                const uint64_t bound = sh.bound, high = bound_of(r, best, t, true);
                if (high != 0 && high >= bound) {
                    const bool all = key_of(best.second, 0) >= bound;
                    const int begin = all ? r.v0 + t : r.v0 + t + (best.vec - r.v0 - t) / (LP_GROUP * THREADS) * LP_GROUP * THREADS;
                    const int end = all ? r.v1 : min(r.v1, begin + LP_GROUP * THREADS);
                    const bool here = r.groups(THREADS) <= LP_STAGES;      // a short part is still in shared memory as a whole
                    for (int v = begin; v < end; v += THREADS) {
                        const uint4 p = here ? ring[v - r.v0] : __ldg(r.vec + v);
                        if (key_of(word_max<T>(max_word<T>(max_word<T>(p.x, p.y), max_word<T>(p.z, p.w))), 0) < bound) continue;
                        float g[Vec16<T>::N];
                        Vec16<T>::unpack(p, g);
#pragma unroll
                        for (int i = 0; i < Vec16<T>::N; ++i) {
                            const uint64_t key = key_of(g[i], (uint32_t)(r.head + v * Vec16<T>::N + i));
                            if (key < bound) continue;
                            const int slot = atomicAdd(&sh.count, 1);
                            if (slot < LpFinish<T, THREADS, TOP>::LIST) sh.list[slot] = key;
                        }
                    }
                }
                __syncwarp();
                bar_arrive<LP_EMPTY>(1);
            }
        }
    }
    if constexpr (CLUSTER) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        cg::this_cluster().sync();
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
    // Values below this count as this with an entropy: their exponential is 0 either way (as in Running).
    __device__ __forceinline__ float floor_value(float m) const { return m - 150.f - fabsf(m) * 0.015625f; }
    // `far`: M is subtracted first.  `floored`: the values have been held to floor_value.
    __device__ __forceinline__ uint64_t pair(float a, float b, bool far, bool floored) const {
        const uint64_t x = far ? add2(pack2(a, b), pack2(-minus, -minus)) : pack2(a, b);
        float d0, d1;
        unpack2(fma2(x, pack2(LOG2E, LOG2E), pack2(-ref, -ref)), d0, d1);
        if (ENTROPY && !floored) { d0 = max_nan(d0, LP_FLOOR); d1 = max_nan(d1, LP_FLOOR); }
        const uint64_t e = mul2(pack2(exp2_fast(d0), exp2_fast(d1)), pack2(scale, scale));
        if (!ENTROPY) return e;
        // d log(2) + H - ln s is log p + H
        const uint64_t lp = fma2(pack2(d0, d1), pack2(LN2, LN2), pack2(shift, shift));
        return mul2(e, fma2(lp, pack2(g_ent, g_ent), pack2(sum, sum)));
    }
    __device__ __forceinline__ float one(float v) const {
        if (nothing) return 0.f;
        float a, b;
        unpack2(pair(v, v, minus != 0.f, false), a, b);
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
    const float low = slope.floor_value(a.stats[2 * row]);
    slope.set(a.stats[2 * row], a.stats[2 * row + 1], sum, ENTROPY ? a.g_entropy[row] : 0.f, ENTROPY ? a.entropy[row] : 0.f);

    int begin, end;      // elements of this segment
    if (same) {
        uint4* out = reinterpret_cast<uint4*>(dx + head);
        uint32_t low_word = 0;
        if constexpr (sizeof(T) == 2) low_word = pack_pair<T>(low, low);
        const auto put = [&](uint4 in, int v, bool far) {
            constexpr bool words = ENTROPY && sizeof(T) == 2;      // two values at once
            if constexpr (words) {
                if (!far) {
                    in.x = max_pair<T>(in.x, low_word); in.y = max_pair<T>(in.y, low_word);
                    in.z = max_pair<T>(in.z, low_word); in.w = max_pair<T>(in.w, low_word);
                }
            }
            float f[VE];
            Vec16<T>::unpack(in, f);
#pragma unroll
            for (int i = 0; i < VE; i += 2) unpack2(slope.pair(f[i], f[i + 1], far, words && !far), f[i], f[i + 1]);
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
    if constexpr (THREADS == 32) __syncwarp(); else __syncthreads();
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
    constexpr int threads = THREADS == 32 ? 128 : LP_TEAM + 32;
    const size_t ring = LpStream<T, THREADS>::RING;
    const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), ring);
    if (st != ADDER_OK) return st;
    if constexpr (CLUSTER) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a.rows * parts));
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = ring;
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
        const long long rows = THREADS == 32 ? (a.rows + 3) / 4 : a.rows, most = (long long)sm_count() * (THREADS == 32 ? 8 : 4);
        // A warp's rows take alike long, so all get as many; CTAs of whole rows spread theirs over all SMs (2048x128000 with entropy, 3.5 rows
        // for each of 592 CTAs: 91 us, 101 with 512 CTAs of 4 rows; 16384x4000 by warps: 37 us, 33 with 1024 CTAs of 4 turns).
        const long long turns = THREADS == 32 ? (rows + most - 1) / most : 1, grid = THREADS == 32 ? (rows + turns - 1) / turns : rows < most ? rows : most;
        kernel<<<(unsigned)grid, threads, ring, s>>>(a);
        return launched();
    }
}

// A warp a row: short rows, and longer ones where there are enough to fill the SMs.  Forward and backward of bf16 with entropy, us by warps and by
// CTAs: 2000x1024 11 and 20, 1184x2048 10 and 16, 1184x4096 14.5 and 16.5, 16384x4000 80 and 141, 3552x8000 37 and 41; on the other side
// 296x2048 10.4 and 8.3, 600x4096 13.4 and 12.4, 1184x8192 18.6 and 17.7 (fp32 29 and 23).
bool warp_rows(long long rows, long long classes) {
    return classes <= 1024 || (classes <= 4096 && rows >= 8LL * sm_count()) || (classes <= 8192 && rows >= 24LL * sm_count());
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
    if (!aligned_to(logits, dtype == ADDER_TYPE_F32 ? 4 : 2) || !aligned_to(targets, 8) || !aligned_to(top_indices, 8) || !aligned_to(stats, 8) ||
        !aligned_to(log_prob, 4) || !aligned_to(entropy, 4) || !aligned_to(top_log_probs, 4))
        return ADDER_ERR_ALIGNMENT;
    const LpFwd a{logits, rows, row_stride, (int)classes, top_k, targets, ignore_index, log_prob, entropy, stats, top_log_probs, top_indices};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        if (warp_rows(rows, classes)) return choose_forward<T, 32, false>(a, 1, s);
        // Few rows leave SMs idle: a row is then split over a cluster of up to 8 CTAs of at least 4096 elements, as long as there are no more than
        // 4 CTAs an SM.  bf16 with entropy by 1, 2, 4 and 8 CTAs, us: 4x32000 6.3, 6.3, 6.3, 5.8 (4 are taken); 64x128000 12.4, 8.3, 8.4, 9.0 (8);
        // 128x50257 8.3, 8.3, 8.6, 12.4 (4); 296x50257 10.4, 12.2, 16.5, 23.4 (2).  From some 2 CTAs an SM on a split costs more than it gives, so
        // the last three take 4 to 18 % more than the best.
        int parts = 1;
        while (parts < 8 && rows * parts * 2 <= sm_count() * 4 && classes >= 8192LL * parts) parts *= 2;
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
    if (!aligned_to(logits, size) || !aligned_to(grad_logits, size) || !aligned_to(targets, 8) || !aligned_to(top_indices, 8) || !aligned_to(stats, 4) ||
        !aligned_to(entropy, 4) || !aligned_to(grad_log_prob, 4) || !aligned_to(grad_entropy, 4) || !aligned_to(grad_top, 4))
        return ADDER_ERR_ALIGNMENT;
    const bool warps = warp_rows(rows, classes);
    // A CTA takes two turns, whose loads and stores overlap (2048x128000 bf16 with an entropy 187 us with one, 161 with two, 164 with three), or
    // one where there would be too few CTAs.
    const long long turn = 256LL * LP_UNROLL * (16 / size), ones = (classes + turn - 1) / turn;
    const long long segments = warps ? 1 : rows * ones >= 8LL * sm_count() ? (ones + 1) / 2 : ones;
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
