// Producers of the paged cache (no reference counterpart: the reference decodes one sequence into
// a contiguous cache).  g4a_paged_qkv_prep does for any number of new tokens of any sequences what
// shaders/fused_per_head_norm_rope.wgsl, per_head_rms_norm_no_weight.wgsl and kv_cache_store.wgsl
// do for one token (src/engine.ts:2061-2091), with the cache row found through the page table;
// g4a_paged_kv_compact moves the rows of an accepted path of drafted tokens together.
#include "g4a_internal.cuh"

namespace {

constexpr int kPrepWarps = 8;

struct PrepParams {
  const float *q, *k, *v;
  const __half *qw, *kw;
  const float* cos_sin;  // [tokens, hd]: cos of the hd/2 pairs, then their sin
  void* q_out;           // f32 or f16 [tokens, nqh, hd]
  __half *k_pages, *v_pages;
  const int *page_table, *token_seq, *slots;
  int batch, page_size, max_pages, num_pages;
  uint32_t tokens;
  int nqh, nkh, hd, heads;  // heads = nqh, + 2 nkh when k and v are given
  size_t q_stride, kv_stride;
  float eps;
  int* err;
};

// The cache row (in units of nkh * hd elements) of a slot, or -1 when it is not to be stored.
__device__ __forceinline__ long long cache_row(const PrepParams& p, int slot, int seq) {
  if (slot < 0) return -1;
  const int j = slot / p.page_size;
  if (j >= p.max_pages) {
    atomicExch(p.err, G4A_DEVERR_SLOT);
    return -1;
  }
  const int page = p.page_table[(size_t)seq * p.max_pages + j];
  if (page < 0 || page >= p.num_pages) {
    atomicExch(p.err, G4A_DEVERR_PAGE);
    return -1;
  }
  return (long long)page * p.page_size + (slot - j * p.page_size);
}

template <int N>
struct alignas(N * 4) FVec {
  float x[N];
};
template <int N>
struct alignas(N * 2) HVec {
  __half x[N];
};

template <int N>
__device__ __forceinline__ void load_f32(const float* src, float (&x)[N]) {
  constexpr int W = N > 4 ? 4 : N;
#pragma unroll
  for (int u = 0; u < N / W; u++) {
    const FVec<W> f = reinterpret_cast<const FVec<W>*>(src)[u];
#pragma unroll
    for (int e = 0; e < W; e++) x[u * W + e] = f.x[e];
  }
}
template <int N>
__device__ __forceinline__ void load_f16(const __half* src, float (&x)[N]) {
  const HVec<N> h = *reinterpret_cast<const HVec<N>*>(src);
#pragma unroll
  for (int e = 0; e < N; e++) x[e] = __half2float(h.x[e]);
}
template <int N>
__device__ __forceinline__ void store_f32(float* dst, const float (&x)[N]) {
  constexpr int W = N > 4 ? 4 : N;
#pragma unroll
  for (int u = 0; u < N / W; u++) {
    FVec<W> f;
#pragma unroll
    for (int e = 0; e < W; e++) f.x[e] = x[u * W + e];
    reinterpret_cast<FVec<W>*>(dst)[u] = f;
  }
}
template <int N>
__device__ __forceinline__ void store_f16(__half* dst, const float (&x)[N]) {
  HVec<N> h;
#pragma unroll
  for (int e = 0; e < N; e++) h.x[e] = __float2half_rn(x[e]);
  *reinterpret_cast<HVec<N>*>(dst) = h;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// y = x w / sqrt(mean(x^2) + eps), then the pairs (p, p + hd/2) turned by the token's angles:
// (a, b) -> (a cos - b sin, a sin + b cos).  v heads are divided only.  Everything is in f32; q leaves
// in f32 or rounded once to f16, k and v rounded once to f16.
// Bound by HBM for many tokens and by latency for few, so a warp takes two neighbouring heads of a
// token, reads its cos / sin row once for both, and issues every load that needs no other one (both
// heads, angles, sequence, slot) before it waits for the first; only the page id has to follow.
// (7,491 tokens of 10 heads of 256 dims, q to f16: 25.4 us, 4.8 TB/s, 0.74 of the measured copy: a warp loads
// once, waits and leaves, 6.3 waves of CTAs, with 62 % of the issue slots used.  One head per warp that first
// looked at the token's sequence 36.  A decode step's token: 2.4 us.)
// VEC > 0: hd = 64 VEC, a lane holds VEC consecutive elements of each half, in vector loads and
// stores (16 bytes at hd >= 256).  VEC = 0: any even hd <= 512 and any alignment, elements
// strided by 32 lanes.
template <int VEC, typename QOut>
__global__ void __launch_bounds__(kPrepWarps * 32) paged_prep_kernel(const PrepParams p) {
  constexpr int N = VEC > 0 ? VEC : 8;  // elements of each half per lane
  const int lane = threadIdx.x & 31;
  const uint32_t pairs = (uint32_t)(p.heads + 1) / 2;
  const uint64_t w = (uint64_t)blockIdx.x * kPrepWarps + (threadIdx.x >> 5);
  const uint32_t tok = (uint32_t)(w / pairs);
  const int head0 = 2 * (int)(w - (uint64_t)tok * pairs);
  const int hd = p.hd, half = hd / 2;
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();
  if (tok >= p.tokens) return;
  // a pair's index of element e of this lane
  auto at = [&](int e) { return VEC > 0 ? lane * N + e : lane + 32 * e; };
  const bool turns = head0 < p.nqh + p.nkh;      // a q or k head among the two
  const bool stores = head0 + 1 >= p.nqh && p.k;  // a k or v head among them (or past the last)
  const int seq = p.token_seq[tok];
  const int slot = stores ? p.slots[tok] : -1;
  float a[2][N], b[2][N], c[N], s[N];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int head = min(head0 + u, p.heads - 1);
    const float* src = head < p.nqh           ? p.q + (size_t)tok * p.q_stride + (size_t)head * hd
                       : head < p.nqh + p.nkh ? p.k + (size_t)tok * p.kv_stride + (size_t)(head - p.nqh) * hd
                                              : p.v + (size_t)tok * p.kv_stride + (size_t)(head - p.nqh - p.nkh) * hd;
    if constexpr (VEC > 0) {
      load_f32<N>(src + lane * N, a[u]);
      load_f32<N>(src + half + lane * N, b[u]);
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const bool in = at(e) < half;
        a[u][e] = in ? src[at(e)] : 0.f;
        b[u][e] = in ? src[half + at(e)] : 0.f;
      }
    }
  }
  if (turns) {
    const float* cs = p.cos_sin + (size_t)tok * hd;
    if constexpr (VEC > 0) {
      load_f32<N>(cs + lane * N, c);
      load_f32<N>(cs + half + lane * N, s);
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const bool in = at(e) < half;
        c[e] = in ? cs[at(e)] : 0.f;
        s[e] = in ? cs[half + at(e)] : 0.f;
      }
    }
  }
  if (seq < 0) return;  // padding: nothing of this token is written
  if (seq >= p.batch) {
    if (lane == 0) atomicExch(p.err, G4A_DEVERR_SLOT);
    return;
  }
  const long long row = stores ? cache_row(p, slot, seq) : -1;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int head = head0 + u;
    if (head >= p.heads) break;
    const bool is_q = head < p.nqh, is_k = !is_q && head < p.nqh + p.nkh;
    if (!is_q && row < 0) continue;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) ss += a[u][e] * a[u][e] + b[u][e] * b[u][e];
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)hd + p.eps);
    float y0[N], y1[N];
    if (is_q || is_k) {
      const __half* wt = is_q ? p.qw : p.kw;
      float wa[N], wb[N];
      if constexpr (VEC > 0) {
        load_f16<N>(wt + lane * N, wa);
        load_f16<N>(wt + half + lane * N, wb);
      } else {
#pragma unroll
        for (int e = 0; e < N; e++) {
          const bool in = at(e) < half;
          wa[e] = in ? __half2float(wt[at(e)]) : 0.f;
          wb[e] = in ? __half2float(wt[half + at(e)]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float x = a[u][e] * wa[e] * inv, y = b[u][e] * wb[e] * inv;
        y0[e] = x * c[e] - y * s[e];
        y1[e] = x * s[e] + y * c[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) y0[e] = a[u][e] * inv, y1[e] = b[u][e] * inv;
    }
    const int kvh = is_q ? 0 : is_k ? head - p.nqh : head - p.nqh - p.nkh;
    __half* kv = (is_k ? p.k_pages : p.v_pages) + ((size_t)(is_q ? 0 : row) * p.nkh + kvh) * hd;
    QOut* qo = reinterpret_cast<QOut*>(p.q_out) + ((size_t)tok * p.nqh + head) * hd;
    if constexpr (VEC > 0) {
      if (!is_q) {
        store_f16<N>(kv + lane * N, y0);
        store_f16<N>(kv + half + lane * N, y1);
      } else if constexpr (sizeof(QOut) == 4) {
        store_f32<N>(qo + lane * N, y0);
        store_f32<N>(qo + half + lane * N, y1);
      } else {
        store_f16<N>(qo + lane * N, y0);
        store_f16<N>(qo + half + lane * N, y1);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) {
        if (at(e) >= half) continue;
        if (!is_q) {
          kv[at(e)] = __float2half_rn(y0[e]);
          kv[half + at(e)] = __float2half_rn(y1[e]);
        } else {
          qo[at(e)] = (QOut)y0[e];
          qo[half + at(e)] = (QOut)y1[e];
        }
      }
    }
  }
}

template <typename QOut>
decltype(&paged_prep_kernel<0, QOut>) pick_prep(uint32_t hd, bool vec) {
  if (vec) switch (hd) {
      case 64: return paged_prep_kernel<1, QOut>;
      case 128: return paged_prep_kernel<2, QOut>;
      case 256: return paged_prep_kernel<4, QOut>;
      case 512: return paged_prep_kernel<8, QOut>;
      default: break;
    }
  return paged_prep_kernel<0, QOut>;
}

// Rows base + path[i] -> base + i of one sequence, as if all were read before any is written
// (a path's later nodes may lie on the places its earlier ones move to).  One CTA per (sequence,
// 128-byte column chunk, tensor): 32 row lanes x 8 chunks of 16 bytes, at most 64 rows, so every
// thread holds its two rows in registers across the one barrier between reads and writes.
// Columns of different CTAs are disjoint, so nothing else has to be ordered.
// Bound by latency, path -> page ids -> rows (1.9 us for 4 rows of 256 dims, 2.6 for 473 rows of 512 dims
// in 64 sequences).
constexpr int kMaxPath = 64;

__global__ void __launch_bounds__(256)
    paged_compact_kernel(__half* k_pages, __half* v_pages, const int* page_table, const int* base_lens,
                         const int* path, const int* path_lens, int max_path, int page_size, int max_pages,
                         int num_pages, int row_chunks, int* err) {
  const int b = blockIdx.x;
  const int col = blockIdx.y * 8 + (threadIdx.x & 7);  // 16-byte chunk of a cache row
  uint4* pool = reinterpret_cast<uint4*>(blockIdx.z ? v_pages : k_pages);
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();
  const int n = path_lens[b], base = base_lens[b];
  if (n <= 0) return;
  const bool first = threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
  if (n > max_path || base < 0) {  // the sequence is left as it was
    if (first) atomicExch(err, G4A_DEVERR_SLOT);
    return;
  }
  auto row_of = [&](long long slot) -> long long {
    if (slot < 0 || slot >= (long long)max_pages * page_size) {
      atomicExch(err, G4A_DEVERR_SLOT);
      return -1;
    }
    const int page = page_table[(size_t)b * max_pages + (int)slot / page_size];
    if (page < 0 || page >= num_pages) {
      atomicExch(err, G4A_DEVERR_PAGE);
      return -1;
    }
    return (long long)page * page_size + (int)slot % page_size;
  };
  uint4 x[2];
  long long dst[2];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int i = (threadIdx.x >> 3) + 32 * u;
    dst[u] = -1;
    if (i >= n || col >= row_chunks) continue;
    const int from = path[(size_t)b * max_path + i];
    if (from == i) continue;
    const long long src = from < 0 ? row_of(-1) : row_of((long long)base + from);
    if (src < 0) continue;
    dst[u] = row_of((long long)base + i);
    if (dst[u] >= 0) x[u] = pool[(size_t)src * row_chunks + col];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; u++)
    if (dst[u] >= 0) pool[(size_t)dst[u] * row_chunks + col] = x[u];
}

g4a_status check_pages(const char* fn, const void* k_pages, const void* v_pages, const void* page_table,
                       uint32_t page_size, uint32_t max_pages, uint32_t num_pages, uint32_t nkh, uint32_t hd) {
  if (!k_pages || !v_pages || !page_table) return g4a_fail(G4A_EINVAL, "%s: null page pool or page_table", fn);
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u)
    return g4a_fail(G4A_EINVAL, "%s: page pools must be 16-byte aligned", fn);
  if (page_size == 0 || max_pages == 0 || num_pages == 0)
    return g4a_fail(G4A_EINVAL, "%s: zero page_size / max_pages_per_seq / num_pages", fn);
  if ((uint64_t)page_size * max_pages > 0x7fffffffull)
    return g4a_fail(G4A_EINVAL, "%s: page_size * max_pages_per_seq exceeds 2^31", fn);
  if (num_pages > 0x7fffffffu) return g4a_fail(G4A_EINVAL, "%s: num_pages exceeds 2^31", fn);
  if (nkh == 0 || nkh > 65536u) return g4a_fail(G4A_EINVAL, "%s: num_kv_heads %u not in [1, 65536]", fn, nkh);
  if (hd == 0 || hd > 512 || (hd % 8) != 0)
    return g4a_fail(G4A_EINVAL, "%s: head_dim %u must be a multiple of 8 in [8, 512]", fn, hd);
  return G4A_OK;
}

}  // namespace

extern "C" {

g4a_status g4a_paged_qkv_prep(g4a_ctx* ctx, const float* q, const float* k, const float* v, const uint16_t* q_norm_w,
                              const uint16_t* k_norm_w, const float* cos_sin, void* q_out, uint32_t q_out_format,
                              uint16_t* k_pages, uint16_t* v_pages, const int32_t* page_table,
                              const int32_t* token_seq, const int32_t* slots, uint32_t num_tokens, uint32_t batch,
                              uint32_t page_size, uint32_t max_pages_per_seq, uint32_t num_pages,
                              uint32_t num_q_heads, uint32_t num_kv_heads, uint32_t head_dim, uint32_t q_row_stride,
                              uint32_t kv_row_stride, float eps) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_paged_qkv_prep";
  if (head_dim == 0 || head_dim > 512 || (head_dim % 8) != 0)
    return g4a_fail(G4A_EINVAL, "%s: head_dim %u must be a multiple of 8 in [8, 512]", fn, head_dim);
  if ((k == nullptr) != (v == nullptr)) return g4a_fail(G4A_EINVAL, "%s: k and v go together (both or neither)", fn);
  if (q_out_format != G4A_ACT_F32 && q_out_format != G4A_ACT_F16)
    return g4a_fail(G4A_EINVAL, "%s: unknown q_out_format %u", fn, q_out_format);
  if (num_tokens > 0x7fffffffu || num_q_heads > 65536u)
    return g4a_fail(G4A_EINVAL, "%s: num_tokens %u or num_q_heads %u too large", fn, num_tokens, num_q_heads);
  const bool kv = k != nullptr;
  if (num_tokens == 0 || (num_q_heads == 0 && !kv)) return G4A_OK;
  if (!cos_sin || !token_seq) return g4a_fail(G4A_EINVAL, "%s: null cos_sin or token_seq", fn);
  if (num_q_heads != 0 && (!q || !q_norm_w || !q_out)) return g4a_fail(G4A_EINVAL, "%s: null q, q_norm_w or q_out", fn);
  if (q_row_stride == 0) q_row_stride = num_q_heads * head_dim;
  if (kv_row_stride == 0) kv_row_stride = num_kv_heads * head_dim;
  if (q_row_stride < (uint64_t)num_q_heads * head_dim)
    return g4a_fail(G4A_EINVAL, "%s: q_row_stride %u below num_q_heads * head_dim", fn, q_row_stride);
  if (kv) {
    if (!k_norm_w || !slots) return g4a_fail(G4A_EINVAL, "%s: null k_norm_w or slots", fn);
    if (g4a_status s = check_pages(fn, k_pages, v_pages, page_table, page_size, max_pages_per_seq, num_pages,
                                   num_kv_heads, head_dim))
      return s;
    if (kv_row_stride < (uint64_t)num_kv_heads * head_dim)
      return g4a_fail(G4A_EINVAL, "%s: kv_row_stride %u below num_kv_heads * head_dim", fn, kv_row_stride);
  }
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  PrepParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.qw = (const __half*)q_norm_w;
  p.kw = (const __half*)k_norm_w;
  p.cos_sin = cos_sin;
  p.q_out = q_out;
  p.k_pages = (__half*)k_pages;
  p.v_pages = (__half*)v_pages;
  p.page_table = page_table;
  p.token_seq = token_seq;
  p.slots = slots;
  p.batch = (int)(batch > 0x7fffffffu ? 0x7fffffffu : batch);
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.tokens = num_tokens;
  p.nqh = (int)num_q_heads;
  p.nkh = (int)num_kv_heads;
  p.hd = (int)head_dim;
  p.heads = p.nqh + (kv ? 2 * p.nkh : 0);
  p.q_stride = q_row_stride;
  p.kv_stride = kv_row_stride;
  p.eps = eps;
  p.err = ctx->dev_err_dev;
  // 16-byte vectors need every row they start from to be aligned; anything else takes the
  // strided instance.
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w |
                         (uintptr_t)cos_sin | (uintptr_t)q_out;
  const bool vec = (ptrs & 15u) == 0 && ((q_row_stride | kv_row_stride) & 3u) == 0;
  const uint64_t warps = (uint64_t)num_tokens * ((uint32_t)(p.heads + 1) / 2);
  const uint64_t blocks = (warps + kPrepWarps - 1) / kPrepWarps;
  if (blocks > 0x7fffffffull) return g4a_fail(G4A_EINVAL, "%s: num_tokens * heads too large", fn);
  g4a_prof_scope ps(ctx, G4A_PROF_PAGED_PREP);
  const cudaError_t e =
      q_out_format == G4A_ACT_F16
          ? g4a_launch(pick_prep<__half>(head_dim, vec), dim3((unsigned)blocks), dim3(kPrepWarps * 32), 0, ctx->stream,
                       true, p)
          : g4a_launch(pick_prep<float>(head_dim, vec), dim3((unsigned)blocks), dim3(kPrepWarps * 32), 0, ctx->stream,
                       true, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch paged_prep_kernel");
  return G4A_OK;
}

g4a_status g4a_paged_kv_compact(g4a_ctx* ctx, uint16_t* k_pages, uint16_t* v_pages, const int32_t* page_table,
                                const int32_t* base_lens, const int32_t* path, const int32_t* path_lens,
                                uint32_t batch, uint32_t max_path, uint32_t page_size, uint32_t max_pages_per_seq,
                                uint32_t num_pages, uint32_t num_kv_heads, uint32_t head_dim) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_paged_kv_compact";
  if (g4a_status s = check_pages(fn, k_pages, v_pages, page_table, page_size, max_pages_per_seq, num_pages,
                                 num_kv_heads, head_dim))
    return s;
  if (max_path > (uint32_t)kMaxPath)
    return g4a_fail(G4A_EINVAL, "%s: max_path %u exceeds %d", fn, max_path, kMaxPath);
  if (batch > 0x7fffffffu) return g4a_fail(G4A_EINVAL, "%s: batch too large", fn);
  if (batch == 0 || max_path == 0) return G4A_OK;
  if (!base_lens || !path || !path_lens) return g4a_fail(G4A_EINVAL, "%s: null base_lens, path or path_lens", fn);
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  const uint32_t row_chunks = num_kv_heads * (head_dim / 8);
  if ((row_chunks + 7) / 8 > 65535u) return g4a_fail(G4A_EINVAL, "%s: num_kv_heads * head_dim too large", fn);
  g4a_prof_scope ps(ctx, G4A_PROF_PAGED_COMPACT);
  const cudaError_t e = g4a_launch(paged_compact_kernel, dim3(batch, (row_chunks + 7) / 8, 2), dim3(256), 0,
                                   ctx->stream, true, (__half*)k_pages, (__half*)v_pages, page_table, base_lens, path,
                                   path_lens, (int)max_path, (int)page_size, (int)max_pages_per_seq, (int)num_pages,
                                   (int)row_chunks, ctx->dev_err_dev);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch paged_compact_kernel");
  return G4A_OK;
}

}  // extern "C"
