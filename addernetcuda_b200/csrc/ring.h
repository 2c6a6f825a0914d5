// A ring of stages whose uses are over in the order in which they began.  Plain C++, so that it is tested without a GPU.
#pragma once

#ifdef __CUDACC__
#define ADDER_RING_FN __host__ __device__ __forceinline__
#else
#define ADDER_RING_FN inline
#endif

namespace adder {

// Waits for the last use of every stage, after `turn` rounds of the ring and `stage` stages more, the oldest first: wait(i, parity) is true once the
// phase of that parity of stage i's barrier is over.  False at the first that does not come, those behind it come later still.
template <int STAGES, class Wait> ADDER_RING_FN bool ring_drain(int stage, int turn, Wait&& wait) {
#ifdef __CUDACC__
#pragma unroll 1
#endif
    for (int j = 0, i = stage; j < STAGES; ++j) {
        const int use = i < stage ? turn : turn - 1;      // -1: the stage has not been used
        if (use >= 0 && !wait(i, (unsigned)(use & 1))) return false;
        if (++i == STAGES) i = 0;
    }
    return true;
}

}  // namespace adder
