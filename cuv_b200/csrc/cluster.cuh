// Thread-block clusters: the hardware's barrier over a cluster's blocks (which are scheduled together, so it always ends), and
// addresses in another block's shared memory.
//
// An arrival releases: what the thread did before it, reads of other blocks' shared memory included, is done for the threads that
// leave the wait.  (A relaxed arrival would order nothing: a block whose shared memory is still being read could end.)
#pragma once
#include "cuvdia_internal.cuh"

namespace cuvdia {

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// the address, in block `rank` of the cluster, of the variable that this block sees at p
__device__ __forceinline__ unsigned in_block(const void* p, unsigned rank) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}

// Dependent launches: a kernel launched with launch_dependent() may start once every block of the kernel before it in the stream
// has called launch_dependents() or ended; what it needs from that kernel it may touch after wait_for_dependencies(), which
// returns when that kernel has ended and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_dependencies() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
inline int launch_dependent(void (*kernel)(P...), unsigned blocks, unsigned threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    return CUVDIA_OK;
}

}  // namespace cuvdia
