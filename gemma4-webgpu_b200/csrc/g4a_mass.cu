// The attention weight that every cached row gets from a chunk of tokens (g4a_paged_key_mass).  No reference
// counterpart.  With the log-sum-exps that the attention has left,
//   mass_r = decay mass_r + sum over the query rows that see r of 2^(scale log2e q k_r - lse log2e),
// so K is read once more and V not at all.  Two kernels:
//  - few query rows to a sequence (decode steps): a warp has 16 keys in registers, as the A operand of mma.sync
//    m16n8k16, 8 query rows are its B operand.  The order of the dims in a product is free, so a lane loads 16
//    consecutive bytes of its rows and uses them as they are: no shared memory for K, 8 or 16 KB in flight for each
//    warp.  The keys of all sequences are dealt in equal parts to one round of CTAs.  Bound by the HBM and by the ends
//    of a step, when a warp multiplies and has nothing under way (24 ragged sequences of up to 16,000 rows of 512 dims:
//    51 us, 5.4 TB/s).  Loading the next step's rows into registers as they are used, or by bulk copies into rings in
//    shared memory, took 129 and 108 us (of 67 then).
//  - chunks: S^T [256 keys x rows] = K Q^T by pairs of CTAs (tcgen05 cta_group::2), a thread is a key and adds up its
//    weights in a register, so nothing is reduced across lanes; the row blocks of a key tile may be cut between
//    pairs, and a last kernel adds the parts up in a fixed order.  Bound by the tensor cores and the exp2 unit
//    together: a block of 128 keys x 128 rows of 256 dims takes 1,024 cycles of either (515 tokens x 8 heads over
//    32,000 rows: 75 us, 0.9 PFLOP/s, the plan and the join with it; tensor pipe 51 % busy).
#include <algorithm>
#include <atomic>

#include "g4a_chunk_pair.cuh"

namespace {

using namespace g4a;
using namespace g4a_chunk;

// ------------------------------------------------------------------------------------ few query rows

constexpr int kFewWarps = 4;
constexpr int kHeld = 4;  // blocks of 8 query rows in shared memory
constexpr int kNoKey = -1 - 0x7fffffff;

// SEG: segments of 32 dims.  Lane 4 g + t holds dims 32 s + 8 t .. + 7 of keys g and g + 8 and of query row g.
// `ctas`: CTAs to be dealt out, 0 (more sequences than threads): gridDim.x for each sequence and kv head.  A sequence's CTAs
// take its steps in turn, so that they share the rows of a window.
template <int SEG>
__global__ void __launch_bounds__(kFewWarps * 32, SEG > 8 ? 2 : 4) mass_few_kernel(const ChunkParams p, int ctas) {
  __shared__ __align__(16) uint4 q_s[kHeld][SEG][32];  // the first query rows as operands: [block][segment][lane]
  __shared__ float z_s[kHeld * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  int b = (int)(blockIdx.y / (unsigned)p.nkh), kvh = (int)(blockIdx.y % (unsigned)p.nkh);
  int part = (int)blockIdx.x, parts = (int)gridDim.x;
  const long long cap = min((long long)p.max_pages * p.page_size, p.mass_stride);
  pdl_wait_primary();
  pdl_launch_dependents();
  if (ctas > 0) {
    const int n = (int)threadIdx.x < p.batch ? (seq_of(p, (int)threadIdx.x, cap).L + 15) / 16 : 0;
    const Deal d = deal_out<kFewWarps * 32>(n, p.nkh, ctas, ctas, kFewWarps, (int)blockIdx.x, -1);
    if (d.b < 0) return;
    b = d.b, kvh = d.local / d.parts, part = d.local - kvh * d.parts, parts = d.parts;
  }
  const Seq s = seq_of(p, b, cap);
  const int base = s.base(), stride = parts * kFewWarps * 16;
  const int* table = p.page_table + (size_t)b * p.max_pages;
  const __half* q = p.q + ((size_t)s.row0 * p.nqh + (size_t)kvh * p.group) * p.hd;
  const float* lse = p.lse + (size_t)s.row0 * p.nqh + (size_t)kvh * p.group;
  float* mass = p.mass + ((size_t)b * p.nkh + kvh) * p.mass_stride;
  const long long rows = (long long)s.T * p.group;
  // 16 bytes of dims d .. of query row r, and its log-sum-exp
  auto query = [&](long long r, int d) {
    if (r >= rows || d >= p.hd) return make_uint4(0, 0, 0, 0);
    const int token = (int)((uint32_t)r / (uint32_t)p.group);
    return __ldg(reinterpret_cast<const uint4*>(q + ((size_t)token * p.nqh + (size_t)(r - (long long)token * p.group)) * p.hd + d));
  };
  auto lse_of = [&](long long r) {
    if (r >= rows) return -INFINITY;
    const int token = (int)((uint32_t)r / (uint32_t)p.group);
    return lse[(size_t)token * p.nqh + (size_t)(r - (long long)token * p.group)];
  };
  const int held = (int)min((rows + 7) / 8, (long long)kHeld);
  for (int i = warp; i < held * SEG; i += kFewWarps) q_s[i / SEG][i % SEG][lane] = query(i / SEG * 8 + g, i % SEG * 32 + t * 8);
  if (threadIdx.x < kHeld * 8) z_s[threadIdx.x] = lse_of(threadIdx.x);
  __syncthreads();
  // the pages of keys g and g + 8, looked up one step ahead
  auto page_of = [&](long long key) { return key < s.L ? table[(uint32_t)key / (uint32_t)p.page_size] : kNoKey; };
  const int k_first = (part * kFewWarps + warp) * 16;
  int pages[2] = {page_of((long long)k_first + g), page_of((long long)k_first + g + 8)};
  for (long long at = k_first; at < s.L; at += stride) {
    const int k0 = (int)at;
    long long off[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t key = (uint32_t)(k0 + g + 8 * h);
      off[h] = (((long long)pages[h] * p.page_size + key % (uint32_t)p.page_size) * p.nkh + kvh) * p.hd;
      if (pages[h] < 0 || pages[h] >= p.num_pages) {
        if (pages[h] != kNoKey) atomicExch(p.err, G4A_DEVERR_PAGE);
        off[h] = -1;
      }
      pages[h] = page_of((long long)key + stride);
    }
    const Tokens see = tokens_of(p, s, k0, 16);
    const bool any = see.first < see.last;
    if (!any && p.decay == 1.f && k0 + 16 <= base) continue;  // nothing changes
    float old[2] = {0.f, 0.f}, sum[2] = {0.f, 0.f};
    uint4 k[2][SEG];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int key = k0 + g + 8 * h;
      if (t == 0 && off[h] >= 0 && key < base && p.decay != 0.f) old[h] = p.decay * mass[key];
#pragma unroll
      for (int e = 0; e < SEG; e++) {
        const int d = e * 32 + t * 8;
        k[h][e] = load_once_if(p.k + off[h] + d, any && off[h] >= 0 && d < p.hd);
      }
    }
    const long long r_end = (long long)see.last * p.group;
    for (long long r0 = any ? (long long)see.first * p.group & ~7ll : r_end; r0 < r_end; r0 += 8) {
      const bool here = r0 < kHeld * 8;
      // The tensor cores cut off what an f32 sum has no bits for, at every step of a chain: 512 dims in one chain lose
      // 4e-6 of a weight on average.  So every 64 dims start from 0, and the sums are added with rounding.
      float c[4] = {0.f, 0.f, 0.f, 0.f}, a[4];
      auto product = [&](int e, const uint4& x) {
        if ((e & 1) == 0) a[0] = a[1] = a[2] = a[3] = 0.f;
        mma_16x8x16(a, k[0][e].x, k[1][e].x, k[0][e].y, k[1][e].y, x.x, x.y);
        mma_16x8x16(a, k[0][e].z, k[1][e].z, k[0][e].w, k[1][e].w, x.z, x.w);
        if ((e & 1) == 1)
#pragma unroll
          for (int i = 0; i < 4; i++) c[i] += a[i];
      };
      if (here) {
#pragma unroll
        for (int e = 0; e < SEG; e++) product(e, q_s[(uint32_t)r0 / 8][e][lane]);
      } else {
        const bool live = r0 + g < rows;
        const int token = live ? (int)((uint32_t)(r0 + g) / (uint32_t)p.group) : 0;
        const __half* row = q + ((size_t)token * p.nqh + (live ? (size_t)(r0 + g - (long long)token * p.group) : 0)) * p.hd;
#pragma unroll
        for (int e = 0; e < SEG; e++) {
          const int d = e * 32 + t * 8;
          product(e, live && d < p.hd ? __ldg(reinterpret_cast<const uint4*>(row + d)) : make_uint4(0, 0, 0, 0));
        }
      }
#pragma unroll
      for (int n = 0; n < 2; n++) {  // query rows r0 + 2 t + n
        const long long r = r0 + 2 * t + n;
        const float z = here ? z_s[r] : lse_of(r);
        if (z == -INFINITY) continue;
        const int pos = base + (int)((uint32_t)r / (uint32_t)p.group);
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (sees(p, pos, k0 + g + 8 * h)) sum[h] += fast_exp2(fmaf(c[2 * h + n], p.scale_log2, -z * kLog2eC));
      }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      if (t == 0 && off[h] >= 0) mass[k0 + g + 8 * h] = old[h] + sum[h];
    }
  }
}

// ------------------------------------------------------------------------------------------- chunks

constexpr int kThreadsM = 512;
constexpr int kTileLog2 = 8, kCtaKeys = 128;  // keys of a tile; of a CTA
constexpr int kWarpK = 8, kWarpQ = 9, kWarpMma = 10, kWarpLse = 11, kWarpTell = 12;
constexpr int kScoreBufs = 4, kLseBufs = 3;

template <int HD>
struct Mc {
  static constexpr int RB = HD > 256 ? 64 : 128;  // query rows of a block, half of them loaded by each CTA
  static constexpr int NC = HD / 64;
  static constexpr int K_CHUNK = kCtaKeys * 128, Q_CHUNK = RB / 2 * 128;
  static constexpr int K_BYTES = NC * K_CHUNK, Q_BYTES = NC * Q_CHUNK;
  static constexpr int NK = HD > 256 ? 1 : 2, NQ = HD <= 128 ? 6 : 3;  // tiles of keys, row blocks in flight
  static constexpr int OFF_Q = NK * K_BYTES;
  static constexpr int OFF_LSE = OFF_Q + NQ * Q_BYTES;            // [kLseBufs][RB] -lse log2e
  static constexpr int OFF_VALID = OFF_LSE + kLseBufs * RB * 4;    // [kLseBufs][4] rows that count
  static constexpr int OFF_SUM = OFF_VALID + kLseBufs * 16;         // [2][128] sums of the second set of warps
  static constexpr int OFF_BAR = OFF_SUM + 2 * kCtaKeys * 4;
  static constexpr int NBARS = 3 * NK + 3 * NQ + 3 * kScoreBufs + 5;
  static constexpr size_t SMEM = (size_t)OFF_BAR + NBARS * 8 + 16;
  static constexpr uint32_t TMEM_COLS = 512;
  static_assert(kScoreBufs * RB <= 512 && SMEM <= 232448, "tile fits");
};

struct MassParams {
  ChunkParams c;
  const Plan* plan;
  const Piece* pieces;
  const int4* seqs;
  const int2* parts;
  float* part;  // [2 * pairs][256]
  int box_k;
  int tokens, heads, head_chunks;  // of a CTA's half block; chunks of heads for a token
};

template <int HD>
__global__ void __launch_bounds__(kThreadsM, 1)
    mass_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq, const MassParams a) {
  using C = Mc<HD>;
  const ChunkParams& p = a.c;
  extern __shared__ __align__(1024) unsigned char smem[];  // (there is no room to align it by hand)
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicExch(p.err, G4A_DEVERR_TMEM);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_landed = bars;                   // [NK] this CTA's keys
  uint64_t* k_ready = k_landed + C::NK;        // [NK] first CTA: of both
  uint64_t* k_free = k_ready + C::NK;          // [NK] the piece's scores done (commit)
  uint64_t* q_landed = k_free + C::NK;         // [NQ] this CTA's half of a row block
  uint64_t* q_ready = q_landed + C::NQ;        // [NQ] first CTA: both
  uint64_t* q_free = q_ready + C::NQ;          // [NQ] scores done (commit)
  uint64_t* s_done = q_free + C::NQ;           // [kScoreBufs] scores (commit), and the block's log-sum-exps (warp 11)
  uint64_t* s_free = s_done + kScoreBufs;      // [kScoreBufs] first CTA: read (4 warps of each)
  uint64_t* lse_free = s_free + kScoreBufs;    // [kLseBufs] read (4 warps)
  uint64_t* sum_full = lse_free + kLseBufs;    // [2] sums of the second set (4 warps)
  uint64_t* sum_free = sum_full + 2;           // [2] read (4 warps)
  uint64_t* all_done = sum_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cta_rank();
  const uint32_t sbase = smem_u32(smem);
  const int half_rows = a.tokens * a.heads;  // rows of a half block that are loaded

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NK; s++) {
      mbar_init(&k_landed[s], 1);
      mbar_init(&k_ready[s], 2);
      mbar_init(&k_free[s], 1);
    }
    for (int s = 0; s < C::NQ; s++) {
      mbar_init(&q_landed[s], 1);
      mbar_init(&q_ready[s], 2);
      mbar_init(&q_free[s], 1);
    }
    for (int s = 0; s < kScoreBufs; s++) {
      mbar_init(&s_done[s], 2);
      mbar_init(&s_free[s], 8);
    }
    for (int s = 0; s < kLseBufs; s++) mbar_init(&lse_free[s], 4);
    for (int s = 0; s < 2; s++) {
      mbar_init(&sum_full[s], 4);
      mbar_init(&sum_free[s], 4);
    }
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmq)) : "memory");
  }
  // rows of a half block that no load fills are zeros for good
  if (half_rows < C::RB / 2) {
    for (int e = threadIdx.x; e < C::NQ * C::Q_BYTES / 16; e += kThreadsM)
      *reinterpret_cast<uint4*>(smem + C::OFF_Q + e * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  __syncwarp();
  if (warp == kWarpMma) {  // one CTA per SM (shared memory), so the allocation never waits
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  pair_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait_primary();
  pdl_launch_dependents();

  const int4 mine = a.plan->pair[blockIdx.x >> 1];
  const int begin = mine.x, end = mine.y;
  bool ok = true;
  uint32_t g = 0, done = 0;  // blocks and pieces so far

  if (warp < 8) {
    // ------------------------------------------------------------------ weights and their sums
    // Warps 0-3 take the even blocks, 4-7 the odd ones; a lane is a key.
    const uint32_t set = (uint32_t)warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int key_in = rank * kCtaKeys + (warp & 3) * 32 + lane;
    float* sums = reinterpret_cast<float*>(smem + C::OFF_SUM);
    for (int i = begin; ok && i < end; i++, done++) {
      const Piece d = a.pieces[i];
      const int key = (d.tile << kTileLog2) + key_in, base = d.L - d.T;
      // the tokens that see the key
      const int see0 = key - base;
      const int see1 = p.window == 0u || (uint32_t)key < p.sinks ? 0x7fffffff : (int)min(0x7fffffffll, (long long)see0 + p.window);
      uint64_t acc[4] = {0, 0, 0, 0};  // pairs of sums
      for (int j = d.j0; j < d.j1; j++, g++) {
        if ((g & 1u) != set) continue;
        const uint32_t buf = g % kScoreBufs;
        ok = warp_wait_own(&s_done[buf], (g / kScoreBufs) & 1u, abort_flag, p.err);
        if (!ok) break;
        tc_fence_after();
        constexpr int kWords = C::RB / 32, kHalfWords = C::RB / 64;
        uint32_t s[2][32];
        tmem_get(lanes + buf * C::RB, s[0]);
        const float* nl = reinterpret_cast<const float*>(smem + C::OFF_LSE) + (g % kLseBufs) * C::RB;
        const uint32_t* valid = reinterpret_cast<const uint32_t*>(smem + C::OFF_VALID + (g % kLseBufs) * 16);
        const int t0 = (d.skip + (a.head_chunks == 1 ? j : j / a.head_chunks)) * 2 * a.tokens;
        uint32_t all = valid[0] & valid[1];
        if (C::RB == 128) all &= valid[2] & valid[3];
        // Where the last columns of a half block are zeros that hold no row (at 3 or 5 heads to a group), an infinite key makes
        // NaN of them, which the weights' selection keeps out.  (The look costs 1 to 2 % there: 5 heads of 256 over 32,000
        // rows 69.5 -> 70.4 us; selecting in every block 2 to 5 %.)
        bool odd = false;
        if (half_rows < C::RB / 2) {
          uint32_t x;
          tmem_get(lanes + buf * C::RB + C::RB - 1, x);
          tmem_wait_ld();
          tmem_landed(x);
          odd = isnan(__uint_as_float(x));
        }
        const bool plain = __all_sync(0xffffffffu, see0 <= t0 && see1 >= t0 + 2 * a.tokens && !odd) && all == 0xffffffffu;
        const uint64_t by = f32x2(p.scale_log2, p.scale_log2);
#pragma unroll
        for (int c = 0; c < kWords; c++) {
          uint32_t(&x)[32] = s[c & 1];
          tmem_wait_ld();
          tmem_landed(x);
          if (c + 1 < kWords) {  // the next word is under way while this one is worked on
            tmem_get(lanes + buf * C::RB + 32u * (c + 1), s[(c + 1) & 1]);
          } else {  // the buffer may be overwritten now
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(map_to(smem_u32(&s_free[buf]), 0));
          }
          uint32_t bits = 0xffffffffu;
          if (!plain) {
            // columns of this word that see the key: those of the tokens [see0, see1)
            const int th = t0 + (c / kHalfWords) * a.tokens, w0 = (c % kHalfWords) * 32;
            const int lo = max(0, min(see0 - th, a.tokens)) * a.heads - w0, hi = max(0, min(see1 - th, a.tokens)) * a.heads - w0;
            const uint32_t from = lo <= 0 ? 0xffffffffu : lo > 31 ? 0u : ~((1u << lo) - 1u);
            const uint32_t to = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u;
            bits = from & to & valid[c];
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 z = *reinterpret_cast<const float4*>(nl + 32 * c + e);
            const float2 u = f32x2_parts(fma_f32x2(f32x2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), by, f32x2(z.x, z.y)));
            const float2 v = f32x2_parts(fma_f32x2(f32x2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), by, f32x2(z.z, z.w)));
            float w[4] = {fast_exp2(u.x), fast_exp2(u.y), fast_exp2(v.x), fast_exp2(v.y)};
            if (!plain) {
#pragma unroll
              for (int k = 0; k < 4; k++)
                if (!((bits >> (e + k)) & 1u)) w[k] = 0.f;
            }
            acc[(e >> 1) & 3] = add_f32x2(acc[(e >> 1) & 3], f32x2(w[0], w[1]));
            acc[((e >> 1) + 1) & 3] = add_f32x2(acc[((e >> 1) + 1) & 3], f32x2(w[2], w[3]));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&lse_free[g % kLseBufs]);
      }
      if (!ok) break;
      const float2 pair_sum = f32x2_parts(add_f32x2(add_f32x2(acc[0], acc[1]), add_f32x2(acc[2], acc[3])));
      const float sum = pair_sum.x + pair_sum.y;
      float* meet = sums + (done & 1u) * kCtaKeys + (warp & 3) * 32 + lane;
      if (set == 1) {
        if (done >= 2) ok = warp_wait_own(&sum_free[done & 1u], ((done >> 1) - 1) & 1u, abort_flag, p.err);
        if (!ok) break;
        *meet = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sum_full[done & 1u]);
      } else {
        ok = warp_wait_own(&sum_full[done & 1u], (done >> 1) & 1u, abort_flag, p.err);
        if (!ok) break;
        const float whole = sum + *meet;
        if (d.slot >= 0) {
          a.part[(size_t)d.slot * (2 * kCtaKeys) + key_in] = whole;
        } else if (key < d.L && row_offset(p, d.b, d.head, key) >= 0) {
          float* at = p.mass + ((size_t)d.b * p.nkh + d.head) * p.mass_stride + key;
          *at = key < base && p.decay != 0.f ? fmaf(p.decay, *at, whole) : whole;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sum_free[done & 1u]);
      }
    }
  } else if (warp == kWarpK) {
    // ------------------------------------------------------------------ keys
    const int boxes = kCtaKeys / a.box_k, ops = boxes * C::NC;
    for (int i = begin; ok && i < end; i++, done++) {
      const Piece d = a.pieces[i];
      const int* table = p.page_table + (size_t)d.b * p.max_pages;
      const uint32_t s = done % C::NK;
      if (done >= (uint32_t)C::NK) ok = warp_wait_own(&k_free[s], (done / C::NK - 1) & 1u, abort_flag, p.err);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&k_landed[s], (uint32_t)C::K_BYTES);
      __syncwarp();
      for (int o = lane; o < ops; o += 32) {
        const int r = o / C::NC, c = o - r * C::NC;
        const int key = (d.tile << kTileLog2) + rank * kCtaKeys + r * a.box_k;
        int page = p.num_pages, row = 0;  // a page that is not there: zeros
        if (key < d.L) {
          const int t = key / p.page_size, id = table[t];
          row = key - t * p.page_size;
          if (id >= 0 && id < p.num_pages) page = id;
        }
        load_box(sbase + s * C::K_BYTES + c * C::K_CHUNK + r * a.box_k * 128, &tmk, 64 * c, d.head, row, page, &k_landed[s]);
      }
    }
    for (uint32_t k = done > (uint32_t)C::NK ? done - C::NK : 0; k < done; k++)
      (void)mbar_wait_bounded(&k_landed[k % C::NK], (k / C::NK) & 1u, p.err, G4A_DEVERR_WAIT_FULL);
  } else if (warp == kWarpQ) {
    // ------------------------------------------------------------------ queries
    for (int i = begin; ok && i < end; i++) {
      const Piece d = a.pieces[i];
      for (int j = d.j0; j < d.j1; j++, g++) {
        const uint32_t s = g % C::NQ;
        if (g >= (uint32_t)C::NQ) ok = warp_wait_own(&q_free[s], (g / C::NQ - 1) & 1u, abort_flag, p.err);
        if (!ok) break;
        const int tb = j / a.head_chunks, hc = j - tb * a.head_chunks;
        const long long token = (long long)d.row0 + ((long long)d.skip + tb) * 2 * a.tokens + rank * a.tokens;
        if (lane == 0) mbar_arrive_expect_tx(&q_landed[s], (uint32_t)(C::NC * half_rows * 128));
        __syncwarp();
        if (lane < C::NC)
          load_box(sbase + C::OFF_Q + s * C::Q_BYTES + lane * C::Q_CHUNK, &tmq, 64 * lane, hc * a.heads, d.head,
                   (int)min(token, (long long)p.tokens), &q_landed[s]);
      }
    }
    for (uint32_t k = g > (uint32_t)C::NQ ? g - C::NQ : 0; k < g; k++)
      (void)mbar_wait_bounded(&q_landed[k % C::NQ], (k / C::NQ) & 1u, p.err, G4A_DEVERR_WAIT_FULL);
  } else if (warp == kWarpMma) {
    // ------------------------------------------------------------------ MMAs of both CTAs
    if (rank == 0) {
      const uint32_t on = elect_one();
      constexpr uint32_t idesc = pair_idesc(C::RB, false);
      const uint64_t dk0 = sw128_desc(sbase, 16, 1024), dq0 = sw128_desc(sbase + C::OFF_Q, 16, 1024);
      for (int i = begin; ok && i < end; i++, done++) {
        const int n = a.pieces[i].j1 - a.pieces[i].j0;
        ok = warp_wait_own(&k_ready[done % C::NK], (done / C::NK) & 1u, abort_flag, p.err);
        const uint64_t dk = dk0 + (uint64_t)(((done % C::NK) * C::K_BYTES) >> 4);
        for (int j = 0; ok && j < n; j++, g++) {
          const uint32_t s = g % C::NQ, buf = g % kScoreBufs;
          if (g >= (uint32_t)kScoreBufs) ok = warp_wait_own(&s_free[buf], (g / kScoreBufs - 1) & 1u, abort_flag, p.err);
          ok = ok && warp_wait_own(&q_ready[s], (g / C::NQ) & 1u, abort_flag, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dq = dq0 + (uint64_t)((s * C::Q_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; kk++) {
            const uint64_t off = (uint64_t)(((kk & 3) * 32) >> 4);
            mma2_ss(on, tmem + buf * C::RB, dk + (uint64_t)(((kk >> 2) * C::K_CHUNK) >> 4) + off,
                    dq + (uint64_t)(((kk >> 2) * C::Q_CHUNK) >> 4) + off, idesc, kk > 0 ? 1u : 0u);
          }
          commit2(on, &s_done[buf]);
          commit2(on, &q_free[s]);
        }
        if (ok) commit2(on, &k_free[done % C::NK]);
      }
      // no MMA may still be running when TMEM is freed, also after an abort
      commit2(on, all_done);
      (void)mbar_wait_bounded(all_done, 0, p.err, G4A_DEVERR_WAIT_MMA);
    }
  } else if (warp == kWarpLse) {
    // ------------------------------------------------------------------ log-sum-exps of the row blocks
    for (int i = begin; ok && i < end; i++) {
      const Piece d = a.pieces[i];
      for (int j = d.j0; j < d.j1; j++, g++) {
        const uint32_t inf = g % kLseBufs;
        const int tb = j / a.head_chunks, hc = j - tb * a.head_chunks;
        const int t0 = (d.skip + tb) * 2 * a.tokens;
        float z[C::RB / 32];
#pragma unroll
        for (int c = 0; c < C::RB / 32; c++) {
          constexpr int kHalfWords = C::RB / 64;
          const int in = (c % kHalfWords) * 32 + lane, tok = t0 + (c / kHalfWords) * a.tokens + in / a.heads;
          const int head = hc * a.heads + in % a.heads;
          z[c] = -INFINITY;
          if (in >= half_rows) z[c] = INFINITY;  // a column that is never anything (its query is zero): weight 0
          else if (tok < d.T && head < p.group)
            z[c] = p.lse[(size_t)(d.row0 + tok) * p.nqh + (size_t)d.head * p.group + head];
        }
        if (g >= (uint32_t)kLseBufs) ok = warp_wait_own(&lse_free[inf], (g / kLseBufs - 1) & 1u, abort_flag, p.err);
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < C::RB / 32; c++) {
          const uint32_t bits = __ballot_sync(0xffffffffu, z[c] != -INFINITY);
          reinterpret_cast<float*>(smem + C::OFF_LSE)[inf * C::RB + 32 * c + lane] = z[c] == -INFINITY ? 0.f : -z[c] * kLog2eC;
          if (lane == 0) reinterpret_cast<uint32_t*>(smem + C::OFF_VALID + inf * 16)[c] = bits;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_done[g % kScoreBufs]);  // (its last use is over: block g - 3 has been read)
      }
    }
  } else if (warp == kWarpTell) {
    // ------------------------------------------------------------------ what has landed in this CTA
    if (lane == 0) {
      for (int i = begin; ok && i < end; i++, done++) {
        ok = wait_own(&k_landed[done % C::NK], (done / C::NK) & 1u, abort_flag, p.err);
        if (!ok) break;
        arrive_at(map_to(smem_u32(&k_ready[done % C::NK]), 0));
        const int n = a.pieces[i].j1 - a.pieces[i].j0;
        for (int j = 0; j < n; j++, g++) {
          ok = wait_own(&q_landed[g % C::NQ], (g / C::NQ) & 1u, abort_flag, p.err);
          if (!ok) break;
          arrive_at(map_to(smem_u32(&q_ready[g % C::NQ]), 0));
        }
      }
    }
  }
  // a warp that gave up stops the partner's waits too (it leaves only through the pair's barrier)
  __syncwarp();
  if (lane == 0 && *abort_flag)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to(smem_u32((const void*)abort_flag), (uint32_t)rank ^ 1u)),
                 "r"(1u)
                 : "memory");
  __syncwarp();
  tc_fence_before();
  pair_sync();
  tc_fence_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
}

// Adds up the parts of the tiles that were cut, and lets the rows fade that no token saw.
__global__ void __launch_bounds__(256) mass_join_kernel(const MassParams a) {
  const ChunkParams& p = a.c;
  pdl_wait_primary();
  pdl_launch_dependents();
  const int b = (int)(blockIdx.y / (unsigned)p.nkh), kvh = (int)(blockIdx.y % (unsigned)p.nkh);
  const Seq s = seq_of(p, b, min((long long)p.max_pages * p.page_size, p.mass_stride));
  const Blocks k = key_tiles_of(p, s, kTileLog2);
  if (a.seqs[b].y < 0) return;  // the call does not fit together
  const int item0 = a.seqs[b].y + kvh * k.count();
  for (int tile = (int)blockIdx.x; (long long)tile << kTileLog2 < s.L; tile += (int)gridDim.x) {
    const int r = (tile << kTileLog2) + (int)threadIdx.x;
    const int e = tile < k.sinks ? tile : tile >= k.window0 && tile < k.window1 ? tile - k.window0 + k.sinks : -1;
    const int2 parts = e >= 0 ? a.parts[item0 + e] : make_int2(0, 0);
    if (parts.y == 1 || (parts.y == 0 && p.decay == 1.f)) continue;
    if ((uint32_t)r >= (uint32_t)s.L || row_offset(p, b, kvh, r) < 0) continue;
    float sum = 0.f;
    // (of the pair that begins the tile, in its place 2 w + 1; of the next ones, in 2 w)
    for (int i = 0; i < parts.y; i++) sum += a.part[(size_t)(2 * (parts.x + i) + (i == 0)) * (2 * kCtaKeys) + threadIdx.x];
    float* at = p.mass + ((size_t)b * p.nkh + kvh) * p.mass_stride + r;
    *at = r < s.base() && p.decay != 0.f ? fmaf(p.decay, *at, sum) : sum;
  }
}

template <int HD>
g4a_status launch_chunk_mass(const char* fn, g4a_ctx* ctx, const ChunkParams& p) {
  using C = Mc<HD>;
  static std::atomic<bool> ready[64];
  if (ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(mass_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(mass_tc_kernel)");
    if (ctx->device < 64) ready[ctx->device].store(true, std::memory_order_release);
  }
  MassParams a = {};
  a.c = p;
  a.heads = std::min(p.group, C::RB / 2);
  a.tokens = C::RB / 2 / a.heads;
  a.head_chunks = (p.group + a.heads - 1) / a.heads;
  a.box_k = std::min(p.page_size & -p.page_size, kCtaKeys);
  CUtensorMap mk, mq;
  if (g4a_status s = g4a_page_map(fn, ctx, &mk, p, p.k, a.box_k)) return s;
  if (g4a_status s = g4a_query_map(fn, ctx, &mq, p, a.heads, a.tokens)) return s;
  const int pairs = std::min(ctx->num_sms / 2, kMaxPairs);
  // key tiles of all sequences, by the room that they have
  const long long rows = std::min<long long>((long long)p.page_size * p.max_pages, p.mass_stride);
  const long long entries = (long long)std::min(p.batch, p.tokens) * ((rows >> kTileLog2) + 2), items = entries * p.nkh;
  if (items > (1 << 26)) return g4a_fail(G4A_EINVAL, "%s: batch * num_kv_heads * rows too large", fn);
  const long long pieces = items + pairs;
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  const size_t n_part = up((size_t)2 * pairs * 2 * kCtaKeys * sizeof(float)), n_plan = up(sizeof(Plan));
  const size_t n_piece = up((size_t)pieces * sizeof(Piece)), n_parts = up((size_t)items * sizeof(int2));
  const size_t n_seq = up((size_t)(p.batch + 1) * sizeof(int4)), n_entry = up((size_t)entries * sizeof(long long));
  if (g4a_status s = g4a_ensure_workspace(ctx, n_part + n_plan + n_piece + n_parts + n_seq + n_entry)) return s;
  char* ws = static_cast<char*>(ctx->workspace);
  PlanParams q = {};
  q.c = p;
  q.pairs = pairs;
  q.halves = 1;
  q.kb_log2 = kTileLog2;
  q.stage_ns = 1.f;
  q.max_entries = entries;
  q.block_tokens = 2 * a.tokens;
  q.head_chunks = a.head_chunks;
  a.part = reinterpret_cast<float*>(ws);
  q.plan = reinterpret_cast<Plan*>(ws += n_part);
  q.pieces = reinterpret_cast<Piece*>(ws += n_plan);
  q.parts = reinterpret_cast<int2*>(ws += n_piece);
  q.seqs = reinterpret_cast<int4*>(ws += n_parts);
  q.entries = reinterpret_cast<long long*>(ws += n_seq);
  a.plan = q.plan;
  a.pieces = q.pieces;
  a.parts = q.parts;
  a.seqs = q.seqs;
  g4a_prof_scope ps(ctx, G4A_PROF_KEY_MASS);
  cudaError_t e = g4a_chunk_plan_launch(ctx, q, true, entries);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_plan_kernel");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kThreadsM);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, mass_tc_kernel<HD>, mk, mq, a);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch mass_tc_kernel");
  const unsigned heads = (unsigned)p.batch * (unsigned)p.nkh;
  const unsigned wide = (unsigned)std::min<long long>((rows + 255) / 256, std::max(1u, 4096u / heads));
  e = g4a_launch(mass_join_kernel, dim3(wide, heads), dim3(256), 0, ctx->stream, true, a);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch mass_join_kernel");
  return G4A_OK;
}

template <int SEG>
g4a_status launch_few(g4a_ctx* ctx, const ChunkParams& p) {
  g4a_prof_scope ps(ctx, G4A_PROF_KEY_MASS);
  const unsigned heads = (unsigned)p.batch * (unsigned)p.nkh;
  const long long rows = std::min<long long>((long long)p.page_size * p.max_pages, p.mass_stride);
  const long long most = (rows + kFewWarps * 16 - 1) / (kFewWarps * 16), round = (SEG > 8 ? 2ll : 4ll) * ctx->num_sms;
  dim3 grid((unsigned)std::min(most, std::max(1ll, 2 * round / heads)), heads);
  int ctas = 0;
  if (p.batch <= kFewWarps * 32) {
    // one round of CTAs, equal parts of the keys; two where the heads are many and the parts so few that one is uneven
    // (64 sequences x 8 heads of 128 dims 123 us with one, 113 with two)
    ctas = (int)std::min(std::max(2ll * heads > round ? 2 * round : round, heads + round / 2), heads * most + heads);
    grid = dim3((unsigned)ctas);
  }
  const cudaError_t e = g4a_launch(mass_few_kernel<SEG>, grid, dim3(kFewWarps * 32), 0, ctx->stream, true, p, ctas);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch mass_few_kernel");
  return G4A_OK;
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
  if ((uint64_t)batch * num_kv_heads > 65535u)
    return g4a_fail(G4A_EINVAL, "%s: batch %u * num_kv_heads %u exceeds 65535", fn, batch, num_kv_heads);
  // By the query rows of a sequence and kv head, on average.  Tiles of 256 keys against 16 keys to a warp, in us:
  //            32 sequences of 8,000 rows, 256 dims    128 dims    16, 512 dims    one of 8,000    32 of 1,000, 256 dims
  //  16 rows   54, 31                                  50, 24      46, 34          14, 8.6         17, 9.0
  //  32 rows   54, 44                                  49, 34      46, 49          14, 10          17, 12
  //  64 rows   54, 111                                 50, 68      46, 104         14, 18          17, 21
  // It is a mean, and the keys are dealt without a look at how many rows read them: 63 sequences with one token and one with 190,
  // 32,000 rows of 256 dims, 8 heads, take 18.9 ms in one call, 164 and 38 us in two.
  const bool few = (uint64_t)num_tokens * (uint64_t)p.group <= 32u * (uint64_t)batch;
  if (head_dim > 256) return few ? launch_few<16>(ctx, p) : launch_chunk_mass<512>(fn, ctx, p);
  if (head_dim > 128) return few ? launch_few<8>(ctx, p) : launch_chunk_mass<256>(fn, ctx, p);
  return few ? launch_few<4>(ctx, p) : launch_chunk_mass<128>(fn, ctx, p);
}
