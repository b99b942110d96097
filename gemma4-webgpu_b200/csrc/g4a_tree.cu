// Attention of drafted tokens over a paged cache (g4a_tree_attn_paged): every token of a tree sees
// the prefix and its own ancestors.  No reference counterpart; the semantics of one token are
// those of shaders/attn_score.wgsl, softmax.wgsl and attn_output.wgsl over the rows it sees.
//
// The T tokens x G q heads that share a kv head are T * G query rows over the same keys, so a
// tile of rows reads a key once for all of them.  One pass over the keys with a running row
// maximum m and sum l: p = 2^(s - m + 7), o = sum p v, l = sum p, both rescaled by 2^(m_old -
// m_new) when m is raised; out = o / l.  Long key ranges are cut over the CTAs; the parts (m, l, o)
// of a tile that several CTAs computed are joined by tree_merge_kernel.
//
// Numbers.  The products run on the tensor cores with f16 operands and f32 sums.  K and V are f16.
// With f32 queries, q and p are each split into two f16 terms (x = hi + lo, lo = f16(x - hi)), 22
// bits together, which is f32's accuracy in all but the last two bits; a query row is scaled by a
// power of two first (its largest element to [2^10, 2^11)) and p carries the factor 2^7, so the
// low terms stay above f16's smallest step (2^-24) for every element that counts.  With f16 queries
// p is rounded once to f16 (the output is f16 too); the sum l is taken over the unrounded p.
//
// This file: the entry point and the join; the attention kernel is in g4a_tree_tc.cu.
#include <algorithm>

#include "g4a_tree.cuh"

namespace {

using namespace g4a;
using namespace g4a_tree;

// Joins the parts of the tiles that were cut between CTAs.  The work is cut into units spread over all
// CTAs.  A thread is a float4 column of a row and a lane over its parts, which it loads four at a time and
// folds with a running maximum; the lanes of a row, if there are several, meet in shared memory.  What
// bounds it is the latency of a unit, cut -> parts -> output, 1 to 2 us cold, not the 5 to 20 MB of parts,
// which lie in the L2: so as many rows to a unit as there are threads for (six parts of 24 tiles with eight
// lanes to a row: five units for each CTA one after another, 18 us; with two lanes 8.5), and many lanes only
// where there are many parts (148 parts of one long context with eight lanes: 9 us, with 32: 5).
constexpr int kMergeThreads = 256;
constexpr int kMergeFly = 4;   // parts of a lane in flight
constexpr int kMaxCuts = 512;  // two for each CTA of the attention kernel

template <bool F32>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeParams p) {
  __shared__ int ends[kMaxCuts];  // running count of units up to and with cut c
  __shared__ int warp_sum[kMergeThreads / 32];
  __shared__ float sm[32][2];
  __shared__ float4 so[kMergeThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait_primary();
  pdl_launch_dependents();
  auto columns_of = [](int parts) { return parts > 32 ? 8 : 32; };
  auto lanes_of = [](int parts) { return parts > 32 ? 32 : parts > 8 ? 8 : parts > 4 ? 2 : 1; };  // over parts
  auto rows_of = [&](int parts) { return kMergeThreads / columns_of(parts) / lanes_of(parts); };  // of a unit
  auto blocks_of = [&](int parts) { return p.hd_pad / 4 / columns_of(parts); };                   // units of a row
  {
    int n[2], incl = 0;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int c = 2 * tid + k;
      n[k] = 0;
      if (c < 2 * p.grid) {
        const int parts = p.cuts[c].parts;
        if (parts > 0) {
          const int rows_per = rows_of(parts);
          n[k] = (p.cuts[c].rows + rows_per - 1) / rows_per * blocks_of(parts);
        }
      }
      incl += n[k];
    }
    const int both = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; w++) incl += warp_sum[w];
    ends[2 * tid] = incl - both + n[0];
    ends[2 * tid + 1] = incl;
    __syncthreads();
  }
  const int total = ends[kMaxCuts - 1];
  const int tile_rows = 1 << p.rows_log2;
  const size_t stride = (size_t)tile_rows * (p.hd_pad + 2);
  for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
    int lo = 0, hi = kMaxCuts - 1;  // the first cut whose end is above the unit
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > unit) hi = mid;
      else lo = mid + 1;
    }
    const Cut cut = p.cuts[lo];
    const int at = unit - (lo ? ends[lo - 1] : 0);
    const int cols = columns_of(cut.parts), pl = lanes_of(cut.parts), blocks = blocks_of(cut.parts);
    const int col = tid & (cols - 1), sub = tid / cols, block = at % blocks;
    const int r = at / blocks * rows_of(cut.parts) + sub / pl, part0 = sub & (pl - 1);
    const int d = (block * cols + col) * 4;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < cut.rows) {
      for (int i0 = part0; i0 < cut.parts; i0 += kMergeFly * pl) {
        float mi[kMergeFly], li[kMergeFly];
        float4 x[kMergeFly];
#pragma unroll
        for (int f = 0; f < kMergeFly; f++) {
          const int i = i0 + f * pl;
          mi[f] = -INFINITY, li[f] = 0.f, x[f] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i >= cut.parts) continue;
          const float* base = p.part + (size_t)(i == 0 ? lo : (lo & ~1) + i * cut.stride) * stride;
          mi[f] = __ldcg(base + (size_t)tile_rows * p.hd_pad + r);
          li[f] = __ldcg(base + (size_t)tile_rows * p.hd_pad + tile_rows + r);
          x[f] = __ldcg(reinterpret_cast<const float4*>(base + (size_t)r * p.hd_pad + d));
        }
        float mn = m;
#pragma unroll
        for (int f = 0; f < kMergeFly; f++) mn = fmaxf(mn, mi[f]);
        const float wo = m == mn ? 1.f : fast_exp2(m - mn);
        m = mn;
        l *= wo;
        o.x *= wo, o.y *= wo, o.z *= wo, o.w *= wo;
#pragma unroll
        for (int f = 0; f < kMergeFly; f++) {
          // a part that saw nothing has weight 0 and sums of 0 (or the NaN of a NaN score, which stays)
          const float w = mi[f] == mn ? 1.f : fast_exp2(mi[f] - mn);
          l = fmaf(w, li[f], l);
          o.x = fmaf(w, x[f].x, o.x);
          o.y = fmaf(w, x[f].y, o.y);
          o.z = fmaf(w, x[f].z, o.z);
          o.w = fmaf(w, x[f].w, o.w);
        }
      }
    }
    if (pl > 1) {  // (the same for the whole unit)
      if (col == 0) sm[sub][0] = m, sm[sub][1] = l;
      so[tid] = o;
      __syncthreads();
    }
    if (part0 == 0 && r < cut.rows && d < p.hd) {
      float lt = l;
      if (pl > 1) {
        float mx = m;
        for (int i = 1; i < pl; i++) mx = fmaxf(mx, sm[sub + i][0]);
        lt = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < pl; i++) {
          const float w = sm[sub + i][0] == mx ? 1.f : fast_exp2(sm[sub + i][0] - mx);
          const float4 x = so[tid + i * cols];
          lt += w * sm[sub + i][1];
          o.x += w * x.x;
          o.y += w * x.y;
          o.z += w * x.z;
          o.w += w * x.w;
        }
      }
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      const int gr = cut.first + r, t = gr / p.group;
      const size_t a = ((size_t)(cut.row0 + t) * p.nqh + cut.kvh * p.group + (gr - t * p.group)) * p.hd + d;
      if constexpr (F32)
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + a) =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      else
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + a) =
            make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    }
    if (pl > 1) __syncthreads();
  }
}

}  // namespace

// The tensor-core kernel (g4a_tree_tc.cu): sets p's tile and launches it.
g4a_status g4a_tree_tc_launch(g4a_ctx* ctx, TreeParams& p, bool f32, long long keys);

extern "C" g4a_status g4a_tree_attn_paged(g4a_ctx* ctx, const void* q, uint32_t format, const uint16_t* k_pages,
                                          const uint16_t* v_pages, const int32_t* page_table, const int32_t* kv_lens,
                                          const int32_t* host_kv_lens, const int32_t* q_indptr,
                                          const uint64_t* tree_mask, uint32_t num_tokens, uint32_t batch,
                                          uint32_t max_tokens, uint32_t page_size, uint32_t max_pages_per_seq,
                                          uint32_t num_pages, uint32_t num_q_heads, uint32_t num_kv_heads,
                                          uint32_t head_dim, float scale, uint32_t sliding_window, void* out) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_tree_attn_paged";
  if (format != G4A_ACT_F32 && format != G4A_ACT_F16) return g4a_fail(G4A_EINVAL, "%s: unknown format %u", fn, format);
  if (num_q_heads == 0 || num_kv_heads == 0 || num_q_heads % num_kv_heads != 0 || num_q_heads > 65536u)
    return g4a_fail(G4A_EINVAL, "%s: num_q_heads %u must be a multiple of num_kv_heads %u", fn, num_q_heads,
                    num_kv_heads);
  if (head_dim == 0 || head_dim > 512 || (head_dim % 8) != 0)
    return g4a_fail(G4A_EINVAL, "%s: head_dim %u must be a multiple of 8 in [8, 512]", fn, head_dim);
  if (max_tokens == 0 || max_tokens > (uint32_t)kMaxTokens)
    return g4a_fail(G4A_EINVAL,
                    "%s: max_tokens %u not in [1, %d] (a longer prompt: several calls, or g4a_prefill_attn over a "
                    "contiguous cache)",
                    fn, max_tokens, kMaxTokens);
  if (batch == 0 || num_tokens == 0) return G4A_OK;
  if (batch > 0x00ffffffu || num_tokens > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: batch %u or num_tokens %u too large", fn, batch, num_tokens);
  if (!q || !k_pages || !v_pages || !page_table || !kv_lens || !q_indptr || !out)
    return g4a_fail(G4A_EINVAL, "%s: null pointer", fn);
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15u)
    return g4a_fail(G4A_EINVAL, "%s: q, out and the page pools must be 16-byte aligned", fn);
  if (page_size == 0 || max_pages_per_seq == 0 || num_pages == 0 || num_pages > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: page_size, max_pages_per_seq or num_pages out of range", fn);
  if ((uint64_t)page_size * max_pages_per_seq > 0x7fff0000ull)
    return g4a_fail(G4A_EINVAL, "%s: page_size * max_pages_per_seq exceeds 2^31", fn);
  // (rows are addressed in 16-byte units of 32 bits)
  if ((uint64_t)num_pages * page_size * num_kv_heads > 0xffffffffull / (head_dim / 8))
    return g4a_fail(G4A_EINVAL, "%s: a page pool of more than 64 GiB", fn);
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  TreeParams p = {};
  p.q = q;
  p.out = out;
  p.k = reinterpret_cast<const __half*>(k_pages);
  p.v = reinterpret_cast<const __half*>(v_pages);
  p.page_table = page_table;
  p.kv_lens = kv_lens;
  p.q_indptr = q_indptr;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.tokens = (int)num_tokens;
  p.batch = (int)batch;
  p.max_tokens = (int)max_tokens;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.nqh = (int)num_q_heads;
  p.nkh = (int)num_kv_heads;
  p.group = (int)(num_q_heads / num_kv_heads);
  p.hd = (int)head_dim;
  p.scale_log2 = scale * kLog2eT;
  p.window = sliding_window;
  p.err = ctx->dev_err_dev;
  const uint64_t cap = (uint64_t)page_size * max_pages_per_seq;
  long long keys = 0;  // rows to be read, over the batch (an upper bound)
  for (uint32_t b = 0; b < batch; b++) {
    uint64_t L = host_kv_lens ? (uint64_t)(host_kv_lens[b] < 0 ? 0 : host_kv_lens[b]) : cap;
    if (L > cap) L = cap;
    if (sliding_window != 0u && L > (uint64_t)sliding_window + max_tokens) L = (uint64_t)sliding_window + max_tokens;
    keys += (long long)L;
  }
  const bool f32 = format == G4A_ACT_F32;
  if (g4a_status s = g4a_tree_tc_launch(ctx, p, f32, keys)) return s;
  if (p.grid > 1) {
    g4a_prof_scope ps(ctx, G4A_PROF_TREE_MERGE);
    const cudaError_t e = g4a_launch(f32 ? tree_merge_kernel<true> : tree_merge_kernel<false>,
                                     dim3(4 * ctx->num_sms), dim3(kMergeThreads), 0, ctx->stream, true, p);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch tree_merge_kernel");
  }
  return G4A_OK;
}
