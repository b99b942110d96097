// A paged cache brought down to a budget of rows (g4a_paged_kv_evict): for each sequence and kv head the first
// rows, the last ones and the heaviest between stay and are moved together.  No reference counterpart.
#include <algorithm>

#include "g4a_internal.cuh"

namespace {

using namespace g4a;

constexpr int kThreadsE = 1024;

struct EvictParams {
  __half *k, *v;
  const int *page_table, *kv_lens;
  float* mass;
  long long mass_stride;
  int batch, budget, sinks, recent, page_size, max_pages, num_pages, nkh, hd;
  int *new_lens, *kept;
  int* idx;  // workspace: [batch, nkh, budget]
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

// One CTA per (sequence, kv head): the border weight by four passes of a radix search, the kept rows' numbers in
// order, then the rows in batches, all of a batch read before any of it is written.
__global__ void __launch_bounds__(kThreadsE) evict_simple_kernel(const EvictParams p) {
  __shared__ int hist[256], warp_sum[32][2], carry[2];
  __shared__ uint32_t prefix_s;
  __shared__ int need_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.nkh, kvh = blockIdx.x % p.nkh;
  const int n = p.kv_lens[b];
  const long long cap = min((long long)p.max_pages * p.page_size, p.mass_stride);
  int* idx = p.idx + ((size_t)b * p.nkh + kvh) * p.budget;
  int* kept = p.kept ? p.kept + ((size_t)b * p.nkh + kvh) * p.budget : nullptr;
  if (kvh == 0 && tid == 0) p.new_lens[b] = n < 0 || n > cap ? n : min(n, p.budget);
  if (n < 0 || n > cap) {
    if (tid == 0) atomicExch(p.err, G4A_DEVERR_TREE);
    return;
  }
  if (n <= p.budget) {
    if (kept)
      for (int i = tid; i < p.budget; i += kThreadsE) kept[i] = i < n ? i : -1;
    return;
  }
  float* mass = p.mass + ((size_t)b * p.nkh + kvh) * p.mass_stride;
  const int first = p.sinks, end = n - p.recent, want = p.budget - p.sinks - p.recent;
  uint32_t prefix = 0, mask = 0;
  int need = want;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreadsE) hist[i] = 0;
    __syncthreads();
    for (int i = first + tid; i < end; i += kThreadsE) {
      const uint32_t o = order_of(mass[i]);
      if ((o & mask) == prefix) atomicAdd(&hist[(o >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255;
      for (; d > 0 && need > hist[d]; d--) need -= hist[d];
      prefix_s = prefix | ((uint32_t)d << shift);
      need_s = need;
    }
    __syncthreads();
    prefix = prefix_s;
    need = need_s;
    mask |= 0xffu << shift;
    __syncthreads();
  }
  // of the rows at the border weight `prefix` the first `need` stay
  if (tid < 2) carry[tid] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += kThreadsE) {
    const int i = i0 + tid;
    bool sure = false, tie = false;
    if (i < n) {
      sure = i < first || i >= end;
      if (!sure && want > 0) {
        const uint32_t o = order_of(mass[i]);
        sure = o > prefix;
        tie = o == prefix;
      }
    }
    const unsigned ts = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) warp_sum[warp][0] = __popc(ts);
    __syncthreads();
    int before = carry[0];
    for (int w = 0; w < warp; w++) before += warp_sum[w][0];
    const bool keep = sure || (tie && before + __popc(ts & ((1u << lane) - 1)) < need);
    const unsigned ks = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_sum[warp][1] = __popc(ks);
    __syncthreads();
    int at = carry[1];
    for (int w = 0; w < warp; w++) at += warp_sum[w][1];
    if (keep) idx[at + __popc(ks & ((1u << lane) - 1))] = i;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < 32; w++) carry[0] += warp_sum[w][0], carry[1] += warp_sum[w][1];
    __syncthreads();
  }
  const int per = p.hd / 8, rows = kThreadsE / per, sub = tid / per, col = tid - sub * per;
  for (int i0 = 0; i0 < p.budget; i0 += rows) {
    const int i = i0 + sub;
    long long src = -1, dst = -1;
    uint4 xk, xv;
    float w = 0.f;
    int from = -1;
    if (sub < rows && i < p.budget) {
      from = idx[i];
      if (kept && col == 0) kept[i] = from;
      if (from != i) {
        src = row_at(p, b, kvh, from);
        dst = row_at(p, b, kvh, i);
        w = mass[from];
        if (src >= 0 && dst >= 0) {
          xk = reinterpret_cast<const uint4*>(p.k + src)[col];
          xv = reinterpret_cast<const uint4*>(p.v + src)[col];
        }
      }
    }
    __syncthreads();
    if (from >= 0 && from != i) {
      if (col == 0) mass[i] = w;
      if (src >= 0 && dst >= 0) {
        reinterpret_cast<uint4*>(p.k + dst)[col] = xk;
        reinterpret_cast<uint4*>(p.v + dst)[col] = xv;
      }
    }
    __syncthreads();
  }
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
  if (g4a_status s = g4a_ensure_workspace(ctx, (size_t)batch * num_kv_heads * budget * sizeof(int))) return s;
  p.idx = static_cast<int*>(ctx->workspace);
  g4a_prof_scope ps(ctx, G4A_PROF_PAGED_EVICT);
  const cudaError_t e =
      g4a_launch(evict_simple_kernel, dim3(batch * num_kv_heads), dim3(kThreadsE), 0, ctx->stream, false, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch evict_simple_kernel");
  return G4A_OK;
}
