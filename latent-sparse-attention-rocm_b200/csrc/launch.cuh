// launch.cuh - launches behind a kernel that is still running, and kernels' attributes (sm_100a).
#pragma once

#include <atomic>

#include "common.cuh"

namespace lsa {

// Launch that may start while the kernel before it drains (programmatic dependent launch): the
// kernel waits (griddepcontrol.wait) before it touches what an earlier kernel writes.
template <typename K, typename... A>
int launch_after(K kern, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? LSA_OK : LSA_ERR_CUDA;
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A kernel's dynamic shared memory (and clusters of more than eight CTAs) allowed, once per device: the
// calls cost about a microsecond each.
template <auto kKernel> bool allow_kernel(int bytes, bool large_clusters = false) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load() & bit) return true;
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    if (large_clusters &&
        cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return false;
    done.fetch_or(bit);
    return true;
}

}  // namespace lsa
