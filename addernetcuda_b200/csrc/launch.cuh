// Launches of kernels whose CTAs share clusters.
#pragma once
#include "kernels.h"

namespace adder {

// Launches `kernel` in clusters of `parts` CTAs (1: none).
template <class Kernel, class... Args> int launch_clusters(Kernel kernel, unsigned grid, unsigned threads, size_t smem, int parts, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        (void)cudaGetLastError();
        return ADDER_ERR_CUDA;
    }
    count_launch();
    return ADDER_OK;
}

}  // namespace adder
