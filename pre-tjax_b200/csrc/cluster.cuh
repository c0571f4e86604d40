// Launching kernels whose blocks work in clusters along x, and reading the other blocks' shared memory.
#pragma once
#include "common.cuh"
#include "tc_common.cuh"

namespace ptj {

// Blocks in consecutive groups of `cluster` (1, 2, 4 or 8; grid.x is a multiple).
template <typename... KArgs, typename... Args>
inline void launch_cluster_k(void (*kern)(KArgs...), dim3 grid, dim3 block, unsigned cluster, size_t smem, cudaStream_t st,
                             Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);  // errors surface through cudaPeekAtLastError
}

// All blocks of the cluster (one: the block) have arrived and see each other's shared memory.
template <int C>
__device__ __forceinline__ void cluster_barrier() {
  if constexpr (C > 1) tc::cluster_sync_all();
  else __syncthreads();
}
template <int C>
__device__ __forceinline__ unsigned cluster_rank() {
  if constexpr (C > 1) return tc::cluster_ctarank();
  else return 0u;
}
// the same variable in the shared memory of block `rank`
template <int C>
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, unsigned rank) {
  if constexpr (C == 1) {
    return *p;
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tc::mapa_shared(tc::smem_u32(p), rank)) : "memory");
    return v;
  }
}
template <int C>
__device__ __forceinline__ double peer_f64(const double* p, unsigned rank) {
  if constexpr (C == 1) {
    return *p;
  } else {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(tc::mapa_shared(tc::smem_u32(p), rank)) : "memory");
    return v;
  }
}

}  // namespace ptj
