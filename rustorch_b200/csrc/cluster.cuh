// Thread-block clusters in the kernels of the 4-bit cache and of eviction: the barrier, and reads of another CTA's shared memory.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace rt {

// Of all threads of the cluster, with release and acquire.  Not the .aligned form, which is undefined for a warp whose threads
// have not met again behind a loop or a branch.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// What lies at `p` in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t remote_address(const void* p, int rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ uint32_t load_remote(const uint32_t* p, int rank) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(remote_address(p, rank)) : "memory");
    return x;
}
__device__ __forceinline__ uint4 load_remote(const uint4* p, int rank) {
    uint4 x;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(remote_address(p, rank))
                 : "memory");
    return x;
}
__device__ __forceinline__ float2 load_remote(const float2* p, int rank) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(remote_address(p, rank)) : "memory");
    return x;
}
__device__ __forceinline__ float4 load_remote(const float4* p, int rank) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(remote_address(p, rank))
                 : "memory");
    return x;
}

}  // namespace rt
