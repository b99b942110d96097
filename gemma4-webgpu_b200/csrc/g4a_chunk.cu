// Attention of a chunk of new tokens of every sequence over a paged cache (g4a_chunk_attn_paged).  No reference
// counterpart; the semantics of one token are those of shaders/attn_score.wgsl, softmax.wgsl and
// attn_output.wgsl over the rows that it sees, with a few first rows beside the window.
#include <cudaTypedefs.h>

#include <cmath>

#include "g4a_chunk_pair.cuh"

using namespace g4a_chunk;

// Tiles of 256 query rows on the tensor cores (g4a_chunk_tc.cu), and few rows from registers (g4a_chunk_few.cu).
g4a_status g4a_chunk_tc_launch(g4a_ctx* ctx, const ChunkParams& p);
g4a_status g4a_chunk_few_launch(g4a_ctx* ctx, const ChunkParams& p);

g4a_status g4a_chunk_params(const char* fn, g4a_ctx* ctx, ChunkParams& p, const uint16_t* q, const uint16_t* k_pages,
                            const uint16_t* v_pages, const int32_t* page_table, const int32_t* kv_lens,
                            const int32_t* q_indptr, uint32_t num_tokens, uint32_t batch, uint32_t page_size,
                            uint32_t max_pages_per_seq, uint32_t num_pages, uint32_t num_q_heads,
                            uint32_t num_kv_heads, uint32_t head_dim, float scale, uint32_t sliding_window,
                            uint32_t sink_tokens) {
  if (num_q_heads == 0 || num_kv_heads == 0 || num_q_heads % num_kv_heads != 0 || num_q_heads > 65536u)
    return g4a_fail(G4A_EINVAL, "%s: num_q_heads %u must be a multiple of num_kv_heads %u", fn, num_q_heads,
                    num_kv_heads);
  if (head_dim == 0 || head_dim > 512 || (head_dim % 8) != 0)
    return g4a_fail(G4A_EINVAL, "%s: head_dim %u must be a multiple of 8 in [8, 512]", fn, head_dim);
  if (!std::isfinite(scale * kLog2eC)) return g4a_fail(G4A_EINVAL, "%s: scale is not finite", fn);
  if (batch > 0x00ffffffu || num_tokens > 0x7fffffffu || (uint64_t)num_tokens * num_q_heads > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: batch %u or num_tokens %u too large", fn, batch, num_tokens);
  if (page_size == 0 || max_pages_per_seq == 0 || num_pages == 0 || num_pages > 0x7fffffffu)
    return g4a_fail(G4A_EINVAL, "%s: page_size, max_pages_per_seq or num_pages out of range", fn);
  if ((uint64_t)page_size * max_pages_per_seq > 0x7fff0000ull)
    return g4a_fail(G4A_EINVAL, "%s: page_size * max_pages_per_seq exceeds 2^31", fn);
  if (batch == 0 || num_tokens == 0) return G4A_OK;
  if (!q || !k_pages || !v_pages || !page_table || !kv_lens || !q_indptr)
    return g4a_fail(G4A_EINVAL, "%s: null pointer", fn);
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15u)
    return g4a_fail(G4A_EINVAL, "%s: q and the page pools must be 16-byte aligned", fn);
  p.q = reinterpret_cast<const __half*>(q);
  p.k = reinterpret_cast<const __half*>(k_pages);
  p.v = reinterpret_cast<const __half*>(v_pages);
  p.page_table = page_table;
  p.kv_lens = kv_lens;
  p.q_indptr = q_indptr;
  p.tokens = (int)num_tokens;
  p.batch = (int)batch;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages_per_seq;
  p.num_pages = (int)num_pages;
  p.nqh = (int)num_q_heads;
  p.nkh = (int)num_kv_heads;
  p.group = (int)(num_q_heads / num_kv_heads);
  p.hd = (int)head_dim;
  p.scale_log2 = scale * kLog2eC;
  p.window = sliding_window;
  p.sinks = sink_tokens;
  p.err = ctx->dev_err_dev;
  return G4A_OK;
}

static g4a_status encode_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const __half* base, const cuuint64_t (&dims)[4],
                             const cuuint64_t (&strides)[3], const cuuint32_t (&box)[4]) {
  if (!ctx->encode_tiled) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || f == nullptr)
      return g4a_fail(G4A_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    ctx->encode_tiled = f;
  }
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  const CUresult r = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ctx->encode_tiled)(
      map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(base), dims, strides, box, steps,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return g4a_fail(G4A_EINVAL, "%s: cuTensorMapEncodeTiled failed (%d)", fn, (int)r);
  return G4A_OK;
}

g4a_status g4a_page_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const ChunkParams& p, const __half* pool,
                        int rows) {
  const cuuint64_t row = (cuuint64_t)p.nkh * p.hd * 2;
  const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.nkh, (cuuint64_t)p.page_size, (cuuint64_t)p.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)p.hd * 2, row, row * p.page_size};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  return encode_map(fn, ctx, map, pool, dims, strides, box);
}

g4a_status g4a_query_map(const char* fn, g4a_ctx* ctx, CUtensorMap* map, const ChunkParams& p, int heads, int tokens) {
  const cuuint64_t head = (cuuint64_t)p.hd * 2;
  const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.group, (cuuint64_t)p.nkh, (cuuint64_t)p.tokens};
  const cuuint64_t strides[3] = {head, head * p.group, head * p.nqh};
  const cuuint32_t box[4] = {64, (cuuint32_t)heads, 1, (cuuint32_t)tokens};
  return encode_map(fn, ctx, map, p.q, dims, strides, box);
}

extern "C" g4a_status g4a_chunk_attn_paged(g4a_ctx* ctx, const uint16_t* q, const uint16_t* k_pages,
                                           const uint16_t* v_pages, const int32_t* page_table, const int32_t* kv_lens,
                                           const int32_t* q_indptr, uint32_t num_tokens, uint32_t batch,
                                           uint32_t page_size, uint32_t max_pages_per_seq, uint32_t num_pages,
                                           uint32_t num_q_heads, uint32_t num_kv_heads, uint32_t head_dim,
                                           float scale, uint32_t sliding_window, uint32_t sink_tokens, float* lse,
                                           uint16_t* out) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_chunk_attn_paged";
  ChunkParams p = {};
  if (g4a_status s = g4a_chunk_params(fn, ctx, p, q, k_pages, v_pages, page_table, kv_lens, q_indptr, num_tokens, batch,
                                      page_size, max_pages_per_seq, num_pages, num_q_heads, num_kv_heads, head_dim,
                                      scale, sliding_window, sink_tokens))
    return s;
  if (batch == 0 || num_tokens == 0) return G4A_OK;
  if (!out) return g4a_fail(G4A_EINVAL, "%s: null pointer", fn);
  if ((uintptr_t)out & 15u) return g4a_fail(G4A_EINVAL, "%s: out must be 16-byte aligned", fn);
  const uint64_t size = (uint64_t)num_tokens * num_q_heads * head_dim;
  if (out < q + size && q < out + size) return g4a_fail(G4A_EINVAL, "%s: out overlaps q", fn);
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  p.lse = lse;
  p.out = reinterpret_cast<__half*>(out);
  // By the query rows of a sequence and kv head, on average (the lengths are on the device).  Tiles of 256 rows against
  // tiles of 8, in us:
  //            32 sequences of 8,000 rows, 256 dims    128 dims    16, 512 dims    one of 8,000    32 of 1,000, 256 dims
  //   8 rows   70, 54                                  62, 33      105, 56         24, 15          28, 18
  //  16 rows   71, 99                                  62, 58      105, 104        24, 24          27, 28
  //  32 rows   73, 190                                 60, 105     107, 197        24, 42          28, 47
  // It is a mean: where the rows are uneven, a long piece among many single tokens is read in tiles of 8 rows that each pass
  // over all of its keys (63 sequences with one token and one with 449, 32,000 rows of 256 dims, one head: 10.7 ms in one
  // call, 342 and 48 us in two; with 190 tokens and 8 heads, which go to tiles of 256, 505 us, and 343 and 57).
  const bool few = (uint64_t)num_tokens * (uint64_t)p.group <= 8u * (uint64_t)batch &&
                   (uint64_t)batch * num_kv_heads <= 65535u;
  return few ? g4a_chunk_few_launch(ctx, p) : g4a_chunk_tc_launch(ctx, p);
}
