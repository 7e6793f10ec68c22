// What kernels on pairs of SMs (`cta_group::2`) share: addresses of the other CTA, cluster barriers, copies that count on the even
// SM's barrier, commits on both.
#pragma once
#include <cuda.h>

#include "tcgen05.cuh"

namespace {

__device__ __forceinline__ uint32_t gp_map(uint32_t addr, int cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
// What a CTA waits for without a limit, and why it ends.  A cluster barrier takes the place of __syncthreads for CTAs that the
// hardware starts together; shared memory of another CTA may only be touched once one has been passed, and no CTA may
// leave before the last access to its own, so an mbarrier with a limit can stand in for neither the first nor the last.  What a kernel has
// to hold to: either every thread of a cluster comes to all of its barriers or none comes to any (a whole cluster may return before the
// first), and all waits in between (rings, accumulators, producers' tails) have a limit, after which they leave their loop.
// Kernels with TMEM: the allocation waits for the other CTA's, right behind the first barrier, and for columns to be free, so a CTA leaves too
// little shared memory on its SM for any other kernel that holds some (each takes 190 KB or more, and gives its columns back on every
// path).  The release waits for the other CTA's, behind a barrier too.
// Not the .aligned forms: the warps come here from loops and branches that their lanes left at different times, and a warp
// that is not converged would count more than once.
__device__ __forceinline__ void gp_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void gp_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void gp_commit(uint32_t bar, uint16_t both) {       // on this barrier of both SMs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(both) : "memory");
}

}  // namespace
