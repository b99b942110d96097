// What the tensor-core kernels of a long-context step share: pairs of CTAs that compute one tile together
// (tcgen05 cta_group::2), their barriers, and the tensor maps of page pools and queries.
#pragma once

#include <cuda.h>

#include "g4a_chunk_plan.cuh"
#include "g4a_tcgen05.cuh"

namespace g4a_chunk {

using namespace g4a;

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ bool try_wait_pair(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait for arrivals of both CTAs.
__device__ __forceinline__ bool wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (try_wait_pair(bar, parity)) return true;
  if (*abort_flag) return false;
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (try_wait_pair(bar, parity)) return true;
    if ((++spins & 63u) == 0u) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > 2000000000ull) {
        *abort_flag = 1;
        if (err) atomicExch(err, G4A_DEVERR_WAIT_MMA);
        return false;
      }
    }
  }
}
// D (+)= A B^T on the pair: M 256, rows 128 c .. of D and A in CTA c, half of B's rows in each.
__device__ __forceinline__ void mma2_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma2_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` of both CTAs when the MMAs issued so far have completed.
__device__ __forceinline__ void commit2(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__host__ __device__ constexpr uint32_t pair_idesc(int n, bool b_mn_major) {
  return (f16_idesc(n, b_mn_major) & 0x00ffffffu) | (uint32_t)(256 >> 4) << 24;  // M 256
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int head, int row, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

}  // namespace g4a_chunk

// Tensor maps: a page pool as {dims, kv heads, rows of a page, pages} in boxes of 64 dims x `rows` rows of one page; the
// queries as {dims, heads of the group, kv heads, tokens} in boxes of 64 dims x `heads` x `tokens`.  Both with the
// 128-byte swizzle; what lies beyond reads as 0.
g4a_status g4a_page_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const g4a_chunk::ChunkParams& p,
                        const __half* pool, int rows);
g4a_status g4a_query_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const g4a_chunk::ChunkParams& p, int heads,
                         int tokens);
