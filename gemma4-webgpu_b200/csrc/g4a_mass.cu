// The attention weight that every cached row gets from a chunk of tokens (g4a_paged_key_mass).  No reference
// counterpart.
#include <algorithm>

#include "g4a_chunk.cuh"

namespace {

using namespace g4a;
using namespace g4a_chunk;

// One warp per (sequence, kv head, row).
__global__ void __launch_bounds__(256) mass_simple_kernel(const ChunkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long cap = min((long long)p.max_pages * p.page_size, p.mass_stride);
  const int b = blockIdx.y / p.nkh, kvh = blockIdx.y % p.nkh;
  const Seq s = seq_of(p, b, cap);
  for (int r = blockIdx.x * 8 + warp; r < s.L; r += gridDim.x * 8) {
    const long long off = row_offset(p, b, kvh, r);
    if (off < 0) continue;
    float sum = 0.f;
    for (int t = max(0, r - s.base()); t < s.T; t++) {
      const int pos = s.base() + t;
      if (!sees(p, pos, r)) continue;
      for (int h = 0; h < p.group; h++) {
        const size_t row = (size_t)(s.row0 + t) * p.nqh + kvh * p.group + h;
        float x = 0.f;
        for (int d = lane; d < p.hd; d += 32) x = fmaf(__half2float(p.q[row * p.hd + d]), __half2float(p.k[off + d]), x);
        for (int w = 16; w >= 1; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        const float lse = p.lse[row];
        if (lse != -INFINITY) sum += exp2f(x * p.scale_log2 - lse * kLog2eC);
      }
    }
    if (lane == 0) {
      float* at = p.mass + ((size_t)b * p.nkh + kvh) * p.mass_stride + r;
      *at = r < s.base() && p.decay != 0.f ? fmaf(p.decay, *at, sum) : sum;
    }
  }
}

}  // namespace

extern "C" g4a_status g4a_paged_key_mass(g4a_ctx* ctx, const uint16_t* q, const float* lse, const uint16_t* k_pages,
                                         const int32_t* page_table, const int32_t* kv_lens, const int32_t* q_indptr,
                                         uint32_t num_tokens, uint32_t batch, uint32_t page_size,
                                         uint32_t max_pages_per_seq, uint32_t num_pages, uint32_t num_q_heads,
                                         uint32_t num_kv_heads, uint32_t head_dim, float scale,
                                         uint32_t sliding_window, uint32_t sink_tokens, float decay, float* mass,
                                         uint64_t mass_stride) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_paged_key_mass";
  if (!(decay >= 0.f && decay <= 1.f)) return g4a_fail(G4A_EINVAL, "%s: decay %g not in [0, 1]", fn, (double)decay);
  if (mass_stride == 0 || mass_stride > 0x7fffffffull)
    return g4a_fail(G4A_EINVAL, "%s: mass_stride %llu out of range", fn, (unsigned long long)mass_stride);
  ChunkParams p = {};
  if (g4a_status s = g4a_chunk_params(fn, ctx, p, q, k_pages, k_pages, page_table, kv_lens, q_indptr, num_tokens, batch,
                                      page_size, max_pages_per_seq, num_pages, num_q_heads, num_kv_heads, head_dim,
                                      scale, sliding_window, sink_tokens))
    return s;
  if (batch == 0 || num_tokens == 0) return G4A_OK;
  if (!lse || !mass) return g4a_fail(G4A_EINVAL, "%s: null pointer", fn);
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  p.lse = const_cast<float*>(lse);
  p.mass = mass;
  p.mass_stride = (long long)mass_stride;
  p.decay = decay;
  g4a_prof_scope ps(ctx, G4A_PROF_KEY_MASS);
  const long long rows = std::min<long long>((long long)page_size * max_pages_per_seq, (long long)mass_stride);
  const cudaError_t e = g4a_launch(mass_simple_kernel, dim3((unsigned)std::min<long long>((rows + 7) / 8, 4096), batch * num_kv_heads),
                                   dim3(256), 0, ctx->stream, false, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch mass_simple_kernel");
  return G4A_OK;
}
