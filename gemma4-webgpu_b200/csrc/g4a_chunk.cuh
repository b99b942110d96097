// What the kernels of a long-context step share (g4a_chunk_attn_paged, g4a_paged_key_mass): the shapes of a call,
// a sequence's place in them, and which rows a token sees.
#pragma once

#include "g4a_internal.cuh"

namespace g4a_chunk {

constexpr float kLog2eC = 1.4426950408889634f;
constexpr float kLn2C = 0.6931471805599453f;

struct ChunkParams {
  const __half* q;  // [tokens, nqh, hd]
  const __half *k, *v;  // page pools [num_pages, page_size, nkh, hd]
  const int *page_table, *kv_lens, *q_indptr;
  int tokens, batch;
  int page_size, max_pages, num_pages;
  int nqh, nkh, group, hd;  // group = nqh / nkh
  float scale_log2;         // scale * log2(e)
  uint32_t window, sinks;
  int* err;
  __half* out;       // attention: [tokens, nqh, hd]
  float* lse;        // attention: written, may be null; masses: read
  float* mass;       // masses: [batch, nkh, mass_stride]
  long long mass_stride;
  float decay;
};

// One sequence: T new tokens (rows row0 .. of q), which are the last of its L rows.  T = 0 and L = 0: nothing to
// do (also for a sequence that does not fit together, which is reported).
struct Seq {
  int row0, T, L;
  __device__ __forceinline__ int base() const { return L - T; }
};

__device__ __forceinline__ Seq seq_of(const ChunkParams& p, int b, long long cap) {
  const int r0 = p.q_indptr[b], r1 = p.q_indptr[b + 1], L = p.kv_lens[b];
  if (r0 < 0 || r1 < r0 || r1 > p.tokens || L < r1 - r0 || L > cap) {
    atomicExch(p.err, G4A_DEVERR_TREE);
    return Seq{0, 0, 0};
  }
  return Seq{r0, r1 - r0, L};
}

// The token of row `pos` sees the rows r <= pos with r >= first_in_window(pos) or r < sinks.
__device__ __forceinline__ int first_in_window(const ChunkParams& p, int pos) {
  return p.window != 0u && (uint32_t)pos >= p.window ? pos + 1 - (int)p.window : 0;
}
__device__ __forceinline__ bool sees(const ChunkParams& p, int pos, int r) {
  return r <= pos && (r >= first_in_window(p, pos) || (uint32_t)r < p.sinks);
}

// Element offset of cache row `key` of sequence b and kv head kvh, or -1 for a bad page id.
__device__ __forceinline__ long long row_offset(const ChunkParams& p, int b, int kvh, int key) {
  const int j = key / p.page_size;
  const int page = p.page_table[(size_t)b * p.max_pages + j];
  if (page < 0 || page >= p.num_pages) {
    atomicExch(p.err, G4A_DEVERR_PAGE);
    return -1;
  }
  return (((long long)page * p.page_size + (key - j * p.page_size)) * p.nkh + kvh) * p.hd;
}

// For the kernels of few query rows, whose operands come straight from global memory.
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes that are read once (in pieces of 64 bytes a row: the L2 fetches their neighbours with them; 64 decode
// sequences 117 -> 111 us).
__device__ __forceinline__ uint4 load_once(const __half* at) {
  uint4 x;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
               : "l"(at));
  return x;
}

// The same, zeros where there is nothing to read, predicated instead of branched to.  The masses of few rows at 512 dims need
// it (24 sequences 61 us with branches, 50 so); attention of few rows takes 109 us with it and 106 with branches.
__device__ __forceinline__ uint4 load_once_if(const __half* at, bool there) {
  uint4 x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(x.x), "=&r"(x.y), "=&r"(x.z), "=&r"(x.w)
      : "l"(at), "r"((int)there));
  return x;
}

// What CTA c does: sequence b, its parts, and kv head and part (kvh * parts + part) in `local`; b < 0: nothing.  A
// sequence of n steps of keys (thread b says how many) has n / q parts, rounded up, `most` at most, with the smallest q
// that lets all have one of the `ctas` CTAs (more than there are heads), and at least `least`.  `own` >= 0 asks for that
// sequence's parts instead.  Up to THREADS sequences.
struct Deal {
  int b, parts, local;
};
template <int THREADS>
__device__ __forceinline__ Deal deal_out(int n, int nkh, int ctas, int most, int least, int c, int own) {
  __shared__ int sums[THREADS / 32], counts[THREADS / 32];
  __shared__ Deal found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int total = __reduce_add_sync(0xffffffffu, n), heads = __reduce_add_sync(0xffffffffu, n > 0 ? nkh : 0);
  if (lane == 0) sums[warp] = total, counts[warp] = heads;
  if (tid == 0) found.b = -1;
  __syncthreads();
  long long all = 0;
  int items = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++) all += sums[i], items += counts[i];
  const long long q = max((all * nkh + (ctas - items) - 1) / (long long)(ctas - items), (long long)least);
  const int parts = n > 0 ? min((int)((n + q - 1) / q), most) : 0;
  int incl = parts * nkh;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++)
    if (i < warp) incl += sums[i];
  const int begin = incl - parts * nkh;
  if (own >= 0 ? tid == own : c >= begin && c < incl) found = Deal{tid, parts, c - begin};
  __syncthreads();
  return found;
}

}  // namespace g4a_chunk

// Checks of the arguments that the two entry points share; fills p but for what each of them adds.
g4a_status g4a_chunk_params(const char* fn, g4a_ctx* ctx, g4a_chunk::ChunkParams& p, const uint16_t* q,
                            const uint16_t* k_pages, const uint16_t* v_pages, const int32_t* page_table,
                            const int32_t* kv_lens, const int32_t* q_indptr, uint32_t num_tokens, uint32_t batch,
                            uint32_t page_size, uint32_t max_pages_per_seq, uint32_t num_pages, uint32_t num_q_heads,
                            uint32_t num_kv_heads, uint32_t head_dim, float scale, uint32_t sliding_window,
                            uint32_t sink_tokens);
