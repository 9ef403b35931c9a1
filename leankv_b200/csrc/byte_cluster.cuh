// Thread-block clusters whose CTAs share the work of some rows and read one another's sums through distributed shared memory.
#pragma once

#include <cstdint>

namespace leankv {
namespace bytes {

constexpr int kMaxCluster = 8;                         // what every device part may hold

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Numbers at a shared address of this CTA's, as the CTA `rank` of the cluster has them there.
__device__ __forceinline__ uint32_t peer(uint32_t at, int rank) {
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    return there;
}
__device__ __forceinline__ float2 peer_f32x2(uint32_t at, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer(at, rank)));
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(uint32_t at, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer(at, rank)));
    return v;
}

}  // namespace bytes
}  // namespace leankv
