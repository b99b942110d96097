// A paged cache brought down to a budget of rows (g4a_paged_kv_evict): for each sequence and kv head the first
// rows, the last ones and the heaviest between stay and are moved together.  No reference counterpart.
// Two kernels, the choice and the move.  One sequence of 131,000 rows of 512 dims to 16,384: 33 us, the latency of the choice
// (24 us by itself with a cold L2) and then the move; 24 sequences x 4 heads of up to 9,000 rows to 4,097: 49 to 52 us,
// 6.0 TB/s, and 61 once on another card.
#include <algorithm>
#include <atomic>

#include "g4a_internal.cuh"

namespace {

using namespace g4a;

constexpr int kThreadsE = 1024;      // of a selecting CTA
constexpr int kBinsE = 2048;
constexpr int kCacheE = 40 * 1024;   // weights that a CTA keeps in shared memory
constexpr int kMaxCluster = 16;
constexpr int kRowsLog2 = 5, kRows = 1 << kRowsLog2;  // rows of a block that is moved at once, one to a lane

struct EvictParams {
  __half *k, *v;
  const int *page_table, *kv_lens;
  float* mass;
  long long mass_stride;
  int batch, budget, sinks, recent, page_size, max_pages, num_pages, nkh, hd;
  int *new_lens, *kept;
  int cap;        // rows that a sequence can have
  int blocks;     // of kRows rows in a budget
  int* idx;       // [batch, nkh, budget] old numbers of the kept rows
  int* rank;      // [batch, nkh, blocks + 1] kept rows before row kRows * block
  int* read;      // [batch, nkh, blocks] 1: the block's rows have been read
  int* ticket;
  int* err;
};

// A weight as a whole number of the same order; +0 and -0 alike, NaN lowest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ long long row_at(const EvictParams& p, int b, int kvh, int row) {
  const int j = row / p.page_size, page = p.page_table[(size_t)b * p.max_pages + j];
  if (page < 0 || page >= p.num_pages) {
    atomicExch(p.err, G4A_DEVERR_PAGE);
    return -1;
  }
  return (((long long)page * p.page_size + (row - j * p.page_size)) * p.nkh + kvh) * p.hd;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_meet(uint32_t ctas) {
  if (ctas == 1) {  // (a meeting of the cluster takes 0.5 us)
    __syncthreads();
    return;
  }
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of CTA `rank`'s shared memory.
__device__ __forceinline__ int peek(const int* at, uint32_t rank) {
  uint32_t addr;
  int x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(at)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

// One cluster of CTAs per (sequence, kv head), each with a slice of the rows between the first and the last ones, in
// order.  The border weight is found digit by digit (11, 11 and 10 bits from the top): every CTA counts its slice,
// all read each other's counts through distributed shared memory.  Then a warp knows how many rows before its own are
// kept, and writes the numbers of its kept rows in order.  Latency: three counts, seven meetings of the cluster, and two
// more ways through the slice.
__global__ void __launch_bounds__(kThreadsE) evict_select_kernel(const EvictParams p) {
  extern __shared__ uint32_t cache[];
  __shared__ int hist[3][kBinsE], sums[2][kBinsE], warp_sum[32], warp_gt[32], warp_tie[32], slice_gt, slice_tie, digit_s, need_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), ctas = cluster_size();
  const int item = (int)(blockIdx.x / ctas), b = item / p.nkh, kvh = item % p.nkh;
  pdl_wait_primary();
  pdl_launch_dependents();
  if (blockIdx.x == 0 && tid == 0) *p.ticket = 0;
  const int n = p.kv_lens[b], budget = p.budget;
  int* kept = p.kept ? p.kept + (size_t)item * budget : nullptr;
  if (kvh == 0 && rank == 0 && tid == 0) p.new_lens[b] = n < 0 || n > p.cap ? n : min(n, budget);
  if (n < 0 || n > p.cap) {  // (the same for the whole cluster, as the next)
    if (tid == 0) atomicExch(p.err, G4A_DEVERR_TREE);
    return;
  }
  if (n <= budget) {
    if (kept)
      for (int i = (int)rank * kThreadsE + tid; i < budget; i += (int)ctas * kThreadsE) kept[i] = i < n ? i : -1;
    return;
  }
  int* idx = p.idx + (size_t)item * budget;
  int* ranks = p.rank + (size_t)item * (p.blocks + 1);
  for (int i = (int)rank * kThreadsE + tid; i < p.blocks; i += (int)ctas * kThreadsE) p.read[(size_t)item * p.blocks + i] = 0;
  const float* mass = p.mass + (size_t)item * p.mass_stride;
  const int first = p.sinks, end = n - p.recent, want = budget - p.sinks - p.recent, middle = end - first;
  // slices of whole warps' rows
  const int per_warp = ((middle + (int)ctas * 32 - 1) / ((int)ctas * 32) + 31) & ~31, slice = per_warp * 32;
  const int at0 = first + (int)rank * slice, count = max(0, min(slice, end - at0));
  const bool cached = count <= kCacheE;
  if (cached) {
#pragma unroll 4
    for (int i = tid; i < count; i += kThreadsE) cache[i] = order_of(mass[at0 + i]);
  }
  auto key_of = [&](int i) { return cached ? cache[i] : order_of(mass[at0 + i]); };
  for (int i = tid; i < 3 * kBinsE; i += kThreadsE) hist[0][i] = 0;
  __syncthreads();
  uint32_t border = 0, mask = 0;
  int need = want;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    int* h = hist[pass];
    for (int i = tid; i < count; i += kThreadsE) {
      const uint32_t o = key_of(i);
      if ((o & mask) == border) atomicAdd(&h[(o >> shift) & (bins - 1)], 1);
    }
    cluster_meet(ctas);
    // every CTA adds up its share of the bins over the cluster, and then all read the sums (every CTA reading all counts
    // took 5.5 us of a pass)
    const int share = (bins + (int)ctas - 1) / (int)ctas, bin0 = (int)rank * share;
    if (ctas > 1) {
      for (int i = tid; i < share && bin0 + i < bins; i += kThreadsE) {
        int x = 0;
#pragma unroll 8
        for (uint32_t r = 0; r < ctas; r++) x += peek(&h[bin0 + i], r);
        sums[pass & 1][i] = x;  // (read by the others before they come to the next pass's first meeting)
      }
      cluster_meet(ctas);
    }
    // bins from the top, two to a thread: the one in which the number of larger ones reaches `need`
    int c[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int bin = kBinsE - 1 - (2 * tid + e);
      if (bin < bins) c[e] = ctas == 1 ? h[bin] : peek(&sums[pass & 1][bin % share], (uint32_t)(bin / share));
    }
    int incl = c[0] + c[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int before = incl - c[0] - c[1] + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (c[e] > 0 && before < need && before + c[e] >= need) digit_s = kBinsE - 1 - (2 * tid + e), need_s = need - before;
      before += c[e];
    }
    __syncthreads();
    if (want > 0) {
      border |= (uint32_t)digit_s << shift;
      need = need_s;
    }
    mask |= (uint32_t)(bins - 1) << shift;
  }
  // ---- of the rows at the border the first `need` stay
  const int w0 = warp * per_warp, w1 = min(count, w0 + per_warp);
  int gt = 0, tie = 0;
  for (int i = w0; i < w1; i += 32) {
    const uint32_t o = i + lane < w1 ? key_of(i + lane) : 0u;
    const bool in = i + lane < w1 && want > 0;
    gt += __popc(__ballot_sync(0xffffffffu, in && o > border));
    tie += __popc(__ballot_sync(0xffffffffu, in && o == border));
  }
  if (lane == 0) warp_gt[warp] = gt, warp_tie[warp] = tie;
  __syncthreads();
  if (warp == 0) {
    const int g = __reduce_add_sync(0xffffffffu, warp_gt[lane]), t = __reduce_add_sync(0xffffffffu, warp_tie[lane]);
    if (lane == 0) slice_gt = g, slice_tie = t;
  }
  cluster_meet(ctas);
  // before this warp: larger ones, and ties (the first `need` of all stay)
  int larger = 0, ties = 0;
  if (lane < (int)rank) larger = peek(&slice_gt, (uint32_t)lane), ties = peek(&slice_tie, (uint32_t)lane);
  if (lane < warp) larger += warp_gt[lane], ties += warp_tie[lane];
  larger = __reduce_add_sync(0xffffffffu, larger);
  ties = __reduce_add_sync(0xffffffffu, ties);
  int at = first + larger + min(ties, need);
  for (int i = w0; i < w1; i += 32) {
    const int row = at0 + i + lane;
    const bool in = i + lane < w1 && want > 0;
    const uint32_t o = in ? key_of(i + lane) : 0u;
    const unsigned tb = __ballot_sync(0xffffffffu, in && o == border), below = (1u << lane) - 1u;
    const bool keep = in && (o > border || (o == border && ties + __popc(tb & below) < need));
    const unsigned kb = __ballot_sync(0xffffffffu, keep);
    const int j = at + __popc(kb & below);
    if (keep) {
      idx[j] = row;
      if (kept) kept[j] = row;
    }
    if (i + lane < w1 && (row & (kRows - 1)) == 0 && row >> kRowsLog2 <= p.blocks) ranks[row >> kRowsLog2] = j;
    at += __popc(kb);
    ties += __popc(tb);
  }
  // the first and the last rows
  for (int i = (int)rank * kThreadsE + tid; i < first + p.recent; i += (int)ctas * kThreadsE) {
    const int row = i < first ? i : end + (i - first), j = i < first ? i : budget - p.recent + (i - first);
    idx[j] = row;
    if (kept) kept[j] = row;
    if ((row & (kRows - 1)) == 0 && row >> kRowsLog2 <= p.blocks) ranks[row >> kRowsLog2] = j;
  }
  cluster_meet(ctas);  // nobody reads this CTA's counts any more
}

// Moves the rows.  Row j comes from row idx[j] >= j, and a block of rows may be written once every row that comes from its
// place has been read; those belong to this block and two before it at most.  So a block is read into shared memory, says
// so, waits for the blocks before it whose rows come from its place, and is written: each byte moves once, all SMs at
// work.  Blocks are taken by ticket, in order, and a block reads before it waits, so those that it waits for always get
// on; the wait is bounded all the same (a block that gives up writes nothing and reports it).  A block is one warp, a lane
// a row, and the copies are bulk ones, so an SM holds 200 KB of rows under way with next to no instructions (256 threads
// with the rows in registers, 128 KB to an SM: 24 and 112 us instead of 22 and 76, with a cold L2, for 131,000 rows to
// 16,384 and for 24 sequences x 4 heads).
__global__ void __launch_bounds__(kRows) evict_move_kernel(const EvictParams p) {
  extern __shared__ __align__(128) unsigned char rows_s[];  // [2][32][hd] f16
  __shared__ uint64_t landed;
  const int lane = threadIdx.x;
  pdl_wait_primary();
  pdl_launch_dependents();
  int ticket = 0;
  if (lane == 0) {
    ticket = atomicAdd(p.ticket, 1);
    mbar_init(&landed, 1);
    fence_mbar_init();
  }
  ticket = __shfl_sync(0xffffffffu, ticket, 0);
  const int item = ticket / p.blocks, block = ticket - item * p.blocks, b = item / p.nkh, kvh = item - b * p.nkh;
  const int n = p.kv_lens[b];
  if (n <= p.budget || n > p.cap) return;
  const int* idx = p.idx + (size_t)item * p.budget;
  const int j0 = block << kRowsLog2, j1 = min(p.budget, j0 + kRows), j = j0 + lane;
  const int from = j < j1 ? idx[j] : j;
  // (the last of them where it was: all are, and nobody waits for them)
  if (__shfl_sync(0xffffffffu, from, j1 - 1 - j0) == j1 - 1) return;
  // the rows whose places lie in this block's come from rows [rank of its begin, rank of its end)
  const int* ranks = p.rank + (size_t)item * (p.blocks + 1);
  const int last = (block + 1) << kRowsLog2 < n ? ranks[block + 1] : p.budget;
  const int wait0 = ranks[block] >> kRowsLog2, wait1 = min(block, ((last - 1) >> kRowsLog2) + 1);
  int* read = p.read + (size_t)item * p.blocks;
  float* mass = p.mass + (size_t)item * p.mass_stride;
  const uint32_t bytes = (uint32_t)p.hd * 2u, mine = smem_u32(rows_s) + (uint32_t)lane * bytes, of_v = kRows * bytes;
  const bool moves = j < j1 && from != j;
  long long src = -1, dst = -1;
  float w = 0.f;
  if (moves) {
    w = mass[from];
    src = row_at(p, b, kvh, from);
    dst = row_at(p, b, kvh, j);
  }
  const bool copies = src >= 0 && dst >= 0;
  const int copied = __popc(__ballot_sync(0xffffffffu, copies));
  if (lane == 0) mbar_arrive_expect_tx(&landed, 2u * bytes * (uint32_t)copied);
  __syncwarp();
  if (copies) {
    const uint32_t bar = smem_u32(&landed);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(mine),
                 "l"(p.k + src), "r"(bytes), "r"(bar)
                 : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(mine + of_v),
                 "l"(p.v + src), "r"(bytes), "r"(bar)
                 : "memory");
  }
  bool ok = mbar_wait_bounded(&landed, 0, p.err, G4A_DEVERR_WAIT_FULL);
  __threadfence();  // the weights have been read too
  ok = __all_sync(0xffffffffu, ok);
  if (lane == 0 && ok) asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(read + block), "r"(1) : "memory");
  if (ok && wait0 + lane < wait1) {
    uint64_t t0 = 0;
    for (uint32_t spins = 1;; spins++) {
      int done;
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(done) : "l"(read + wait0 + lane) : "memory");
      if (done) break;
      if ((spins & 63u) != 0u) continue;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > 2000000000ull) {
        ok = false;
        atomicExch(p.err, G4A_DEVERR_WAIT_FULL);
        break;
      }
    }
  }
  if (!__all_sync(0xffffffffu, ok)) return;
  if (copies) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.k + dst), "r"(mine), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.v + dst), "r"(mine + of_v), "r"(bytes)
                 : "memory");
  }
  if (moves) mass[j] = w;
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

}  // namespace

extern "C" g4a_status g4a_paged_kv_evict(g4a_ctx* ctx, uint16_t* k_pages, uint16_t* v_pages, const int32_t* page_table,
                                         const int32_t* kv_lens, float* mass, uint64_t mass_stride, uint32_t batch,
                                         uint32_t budget, uint32_t sink_tokens, uint32_t recent_tokens,
                                         uint32_t page_size, uint32_t max_pages_per_seq, uint32_t num_pages,
                                         uint32_t num_kv_heads, uint32_t head_dim, int32_t* new_lens, int32_t* kept) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_paged_kv_evict";
  if (num_kv_heads == 0 || num_kv_heads > 65536u)
    return g4a_fail(G4A_EINVAL, "%s: num_kv_heads %u not in [1, 65536]", fn, num_kv_heads);
  if (head_dim == 0 || head_dim > 512 || (head_dim % 8) != 0)
    return g4a_fail(G4A_EINVAL, "%s: head_dim %u must be a multiple of 8 in [8, 512]", fn, head_dim);
  if (budget == 0 || budget > 0x7fffffffu) return g4a_fail(G4A_EINVAL, "%s: budget %u out of range", fn, budget);
  if ((uint64_t)sink_tokens + recent_tokens > budget)
    return g4a_fail(G4A_EINVAL, "%s: sink_tokens %u and recent_tokens %u exceed the budget of %u rows", fn, sink_tokens,
                    recent_tokens, budget);
  if (page_size == 0 || max_pages_per_seq == 0 || num_pages == 0 || num_pages > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: page_size, max_pages_per_seq or num_pages out of range", fn);
  if ((uint64_t)page_size * max_pages_per_seq > 0x7fff0000ull)
    return g4a_fail(G4A_EINVAL, "%s: page_size * max_pages_per_seq exceeds 2^31", fn);
  if (mass_stride == 0 || mass_stride > 0x7fffffffull)
    return g4a_fail(G4A_EINVAL, "%s: mass_stride %llu out of range", fn, (unsigned long long)mass_stride);
  if (batch > 0x00ffffffu || (uint64_t)batch * num_kv_heads > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: batch %u too large", fn, batch);
  if (batch == 0) return G4A_OK;
  if (!k_pages || !v_pages || !page_table || !kv_lens || !mass || !new_lens)
    return g4a_fail(G4A_EINVAL, "%s: null pointer", fn);
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u)
    return g4a_fail(G4A_EINVAL, "%s: the page pools must be 16-byte aligned", fn);
  if (new_lens < kv_lens + batch && kv_lens < new_lens + batch)
    return g4a_fail(G4A_EINVAL, "%s: new_lens overlaps kv_lens", fn);
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  EvictParams p = {};
  p.k = reinterpret_cast<__half*>(k_pages);
  p.v = reinterpret_cast<__half*>(v_pages);
  p.page_table = page_table;
  p.kv_lens = kv_lens;
  p.mass = mass;
  p.mass_stride = (long long)mass_stride;
  p.batch = (int)batch;
  p.budget = (int)budget;
  p.sinks = (int)sink_tokens;
  p.recent = (int)recent_tokens;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.nkh = (int)num_kv_heads;
  p.hd = (int)head_dim;
  p.new_lens = new_lens;
  p.kept = kept;
  p.err = ctx->dev_err_dev;
  const uint64_t cap = std::min<uint64_t>((uint64_t)page_size * max_pages_per_seq, mass_stride);
  const long long items = (long long)batch * num_kv_heads;
  p.cap = (int)cap;
  const bool any = budget < cap;  // whether a sequence can have more rows than the budget
  p.blocks = any ? (int)(((long long)p.budget + kRows - 1) >> kRowsLog2) : 1;
  if (any && items * (p.blocks + 1ll) > 0x7fffffffll) return g4a_fail(G4A_EINVAL, "%s: batch * num_kv_heads * budget too large", fn);
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const size_t n_idx = any ? up((size_t)items * budget * sizeof(int)) : 0, n_block = any ? up((size_t)items * (p.blocks + 1) * sizeof(int)) : 0;
  if (g4a_status s = g4a_ensure_workspace(ctx, 256 + n_idx + 2 * n_block)) return s;
  char* ws = static_cast<char*>(ctx->workspace);
  p.ticket = reinterpret_cast<int*>(ws);
  p.idx = reinterpret_cast<int*>(ws += 256);
  p.rank = reinterpret_cast<int*>(ws += n_idx);
  p.read = reinterpret_cast<int*>(ws += n_block);
  static std::atomic<bool> ready[64];
  const size_t smem = kCacheE * sizeof(uint32_t);
  if (ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)  // 64 KB: 32 rows of 512 dims, K and V
      e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kRows * 512 * 2);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(evict kernels)");
    if (ctx->device < 64) ready[ctx->device].store(true, std::memory_order_release);
  }
  // CTAs of a cluster: slices of some 4,096 rows, as far as there are SMs
  int ctas = 1;
  while (ctas < kMaxCluster && cap > (uint64_t)ctas * 4096 && 2 * ctas * items <= ctx->num_sms) ctas *= 2;
  if (items * ctas > 0x7fffffffll) return g4a_fail(G4A_EINVAL, "%s: batch * num_kv_heads too large", fn);
  g4a_prof_scope ps(ctx, G4A_PROF_PAGED_EVICT);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * ctas));
  cfg.blockDim = dim3(kThreadsE);
  cfg.dynamicSmemBytes = any ? std::min(smem, (size_t)((cap / ctas + 1024 + 31) & ~31ull) * sizeof(uint32_t)) : 0;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch evict_select_kernel");
  if (any) {
    e = g4a_launch(evict_move_kernel, dim3((unsigned)(items * p.blocks)), dim3(kRows), (size_t)2 * kRows * p.hd * 2, ctx->stream,
                   true, p);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch evict_move_kernel");
  }
  return G4A_OK;
}
