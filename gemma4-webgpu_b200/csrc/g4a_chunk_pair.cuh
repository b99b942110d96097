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
// Arrivals on a barrier of either CTA.  publish_at is for a thread whose stores to shared memory the other CTA's waits have
// to see: it drains all that the thread has under way, 1,300 to 1,800 cycles.  arrive_at orders what is not stored by
// plain stores: TMEM accesses (behind a tcgen05 fence) and copies whose arrival this thread has seen.
__device__ __forceinline__ void publish_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
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
// Bounded waits: for arrivals of both CTAs, of this one alone.  The timer is looked at only after a number of tries
// (reading it takes longer than most waits).
template <bool PAIR>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  uint64_t t0 = 0;
  for (uint32_t spins = 1;; spins++) {
    if (PAIR ? try_wait_pair(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if ((spins & 63u) == 0u) {
      if (*abort_flag) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > 2000000000ull) {
        *abort_flag = 1;
        if (err) atomicExch(err, G4A_DEVERR_WAIT_MMA);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  return wait_bar<true>(bar, parity, abort_flag, err);
}
__device__ __forceinline__ bool wait_own(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  return wait_bar<false>(bar, parity, abort_flag, err);
}
__device__ __forceinline__ bool warp_wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  return __all_sync(0xffffffffu, wait_pair(bar, parity, abort_flag, err));
}
__device__ __forceinline__ bool warp_wait_own(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  return __all_sync(0xffffffffu, wait_own(bar, parity, abort_flag, err));
}

// D (+)= A B^T on the pair: M 256, rows 128 c .. of D and A in CTA c, half of B's rows in each.  Issued by the lane for
// which `on` is not 0; the instructions are predicated, not branched to, so that the warp's control flow stays uniform
// and the descriptors in uniform registers (11 cycles to issue one instead of 45, and 80 beside busy softmax warps).
__device__ __forceinline__ void mma2_ss(uint32_t on, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma2_ts(uint32_t on, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// Arrive on `bar` of both CTAs when the MMAs issued so far have completed.
__device__ __forceinline__ void commit2(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3), "r"(on)
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

// Two f32 in one instruction.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

}  // namespace g4a_chunk

// Tensor maps: a page pool as {dims, kv heads, rows of a page, pages} in boxes of 64 dims x `rows` rows of one page; the
// queries as {dims, heads of the group, kv heads, tokens} in boxes of 64 dims x `heads` x `tokens`.  Both with the
// 128-byte swizzle; what lies beyond reads as 0.
g4a_status g4a_page_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const g4a_chunk::ChunkParams& p,
                        const __half* pool, int rows);
g4a_status g4a_query_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const g4a_chunk::ChunkParams& p, int heads,
                         int tokens);
