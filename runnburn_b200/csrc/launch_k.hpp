// How every kernel of the library is launched: one wrapper around cudaLaunchKernelEx, with or without clusters.
#pragma once
#include "state.hpp"

namespace rnb {

// Programmatic dependent launch (off with RNB_B200_PDL=0): kernels overlap their weight
// prefetch and set-up with the tail of the previous kernel.  EVERY kernel launched through
// launch_k must execute pdl_wait() before it touches memory another kernel wrote: a kernel
// that skips it neither waits for its predecessor nor orders its successor behind it.  And it
// must reach that memory through plain pointers and loads: __restrict__, __ldg and ld.global.nc
// let the compiler load ahead of the wait (pdl_wait in common.cuh has the rule).
bool use_pdl();

// Kernels launched by this library so far (callers take differences).
inline uint64_t &launch_count() {
    static uint64_t n = 0;
    return n;
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                            cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    if (use_pdl()) {
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
    if (e == cudaSuccess) launch_count()++;
    return e;
}

// The same launch in thread-block clusters.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_k_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, dim3 cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster.x;
    attr[0].val.clusterDim.y = cluster.y;
    attr[0].val.clusterDim.z = cluster.z;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
    if (e == cudaSuccess) launch_count()++;
    return e;
}

}  // namespace rnb
