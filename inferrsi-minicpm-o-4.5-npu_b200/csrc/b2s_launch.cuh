// Host side: kernel launches with programmatic stream serialisation, with or without a cluster.
#pragma once

#include <cuda_runtime.h>
#include <string.h>

namespace b2s {

template <typename... P, typename... A>
cudaError_t launch_cluster(void (*kernel)(P...), dim3 grid, int cluster, int threads, uint32_t smem, void* stream,
                           A... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem, void* stream, A... args) {
    return launch_cluster(kernel, grid, 1, threads, smem, stream, args...);
}

}  // namespace b2s
