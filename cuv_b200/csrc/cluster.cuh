// Thread-block clusters: the hardware's barrier over a cluster's blocks (which are scheduled together, so it always ends), and
// addresses in another block's shared memory.
#pragma once
#include "cuvdia_internal.cuh"

namespace cuvdia {

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
// for blocks that only tell each other how far they are, with nothing written to be seen
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// the address, in block `rank` of the cluster, of the variable that this block sees at p
__device__ __forceinline__ unsigned in_block(const void* p, unsigned rank) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}

}  // namespace cuvdia
