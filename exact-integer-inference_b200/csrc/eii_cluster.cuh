// Thread-block clusters, asynchronous copies to shared memory, and exact 64-bit sums over a warp.
#pragma once
#include <cstdint>

#include "eii_ptx.cuh"

namespace eii {

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t remote_smem(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int32_t ld_remote32(uint32_t a) {
    int32_t v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ int64_t ld_remote64(uint32_t a) {
    int64_t v;
    asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
// Sum of a non-negative v over the warp, in pieces of 24 bits and the rest.  Exact where every lane's v (one thread's,
// warp's or block's part) is below 2^51, so that 32 upper pieces stay in 32 bits; the parts here are below
// 2^47, their sum may be more: 2^18 weights of 2^30 make 2^48.
__device__ __forceinline__ uint64_t warp_sum47(uint64_t v) {
    const uint32_t lo = __reduce_add_sync(~0u, static_cast<uint32_t>(v) & 0xFFFFFFu);
    const uint32_t hi = __reduce_add_sync(~0u, static_cast<uint32_t>(v >> 24));
    return (static_cast<uint64_t>(hi) << 24) + lo;
}
// The same of a signed |v| < 2^50.
__device__ __forceinline__ int64_t warp_sum_signed(int64_t v) {
    const uint32_t lo = __reduce_add_sync(~0u, static_cast<uint32_t>(v) & 0xFFFFFFu);
    const int32_t hi = __reduce_add_sync(~0u, static_cast<int32_t>(v >> 24));
    return (static_cast<int64_t>(hi) << 24) + lo;
}

}  // namespace eii
