// Rows of logits on their way through shared memory, as the operators on them read them.  A call's arguments `a` name the logits x, the rows, the
// elements from row to row (stride) and the classes.
#pragma once
#include "softmax.cuh"

namespace adder {

constexpr int LP_TEAM = 256;                    // threads that stream one row; a CTA has one warp more, which finishes rows
constexpr int LP_GROUP = 4, LP_STAGES = 2;      // vectors of a thread that are taken together, groups of them on their way or in use

// A row as a team sees it: aligned vectors v0 to v1 - 1 (shared out over the cluster), and up to VE - 1 single elements before and
// behind all vectors, which are rank 0's.
template <class T> struct LpRow {
    static constexpr int VE = Vec16<T>::N;
    const T* x;
    const uint4* vec;
    int head, nvec, singles, v0, v1;

    template <class A> __device__ __forceinline__ void set(const A& a, long long row, int rank, int parts) {
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

    template <class A> __device__ __forceinline__ void set_row(const A& a, int t, int rank, int parts) {
        LpRow<T> r;
        r.set(a, row, rank, parts);
        src = r.vec + r.v0 + t;
        left = r.v1 - r.v0 - t;
        groups = r.groups(THREADS);
    }
    template <class A> __device__ __forceinline__ void issue(const A& a, int t, int rank, int parts) {
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

}  // namespace adder
