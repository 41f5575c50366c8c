// Pieces of the CTA-pair kernels (rtb_pairgemm.cu, rtb_mxgemm.cu): addresses and
// barriers of the pair, loads and commits that signal both CTAs.
#pragma once
#include "rtb_blockgemm.cuh"

namespace rtb {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address in CTA `rank` of the cluster of this CTA's shared address.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// Arrival on a barrier of the pair.  What it orders is TMEM traffic (the
// loads have been waited for, tcgen05.fence on both sides) and no generic
// memory, so CTA scope is enough: a cluster-scope release is a memory barrier
// that also waits for the scale loads in flight (it took two thirds of the
// epilogue's time), a cluster-scope acquire drops them from L1.
__device__ __forceinline__ void arrive_pair(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A tiled load into this CTA that completes on a barrier of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                                 int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
// Arrive on both CTAs' barrier at this offset once the MMAs issued so far are
// done.
__device__ __forceinline__ void commit_pair_e(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t.reg .b16 m;\n\t"
      "mov.b16 m, 3;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], m;\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

}  // namespace rtb
