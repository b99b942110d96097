// The tensor-core kernel of g4a_chunk_attn_paged (tcgen05 / TMEM on pairs of CTAs) and the join of cut tiles.
//
// Rows of a tile are the T tokens x G q heads that share a kv head, 256 of them: a pair of CTAs computes them
// together with tcgen05.mma.cta_group::2 (M 256), 128 rows in each CTA, so a key that is loaded serves 256 rows and
// each CTA holds only half of every K and V block: with 128 rows to a K and V block of its own, each SM would ask
// the L2 for 64 bytes per cycle at the tensor cores' full rate, which is all that an SM gets.
//   S [256 x KB]  = Q K^T    A = Q (each CTA's 128 rows), B = K block, half of its keys in each CTA
//   O [256 x HDV] += P V     A = P from TMEM, where the scores were, B = V block, half of its dims in each CTA
// One pass over the keys with a running row maximum m and sum l: p = 2^(s - m), rounded to f16 for the product with V
// and summed unrounded; m follows the maximum lazily, and O is rescaled only when it is raised.  KB is 128 keys.
// Heads of more than 256 dims: O takes 256 TMEM columns, so the dims of V are halved between two pieces of work, each
// with the scores of its own (3/2 of the products, but nothing to be exchanged, where two CTAs that split the dims
// have to add each other's partial scores); 64 keys, for Q takes 128 KB.
//
// What bounds it.  256 dims: the clock that the power limit leaves (512 tokens x 8 heads over 131,000 rows: 594,000 cycles with
// the tensor pipe 79 % busy; 458 us, 1.2 PFLOP/s, in calls for seconds on end at 1,000 W, 388 in short bursts).  512 dims: Q
// comes from shared memory for every 64 keys (1,536 cycles for 1,024 of products), beside the half of the
// scores that is computed twice (1,001 tokens x 8 heads over 20,003 rows: 450 us, 0.71 PFLOP/s, tensor pipe 64 % busy).
// 128 dims: the softmax of a stage, about 2,500 cycles for 1,024 of MMAs (six ragged pieces: 197 us, 0.66 PFLOP/s, 39 %): the
// exp2 unit's 1,024, and waits, scores from TMEM, maxima and their exchange, which nothing overlaps.  Two sets of
// warps that take whole stages in turn (237 us), or the next stage's maxima ahead of this one's weights (226), read the
// scores twice and were slower.
//
// Warps of a CTA (16):
//   0-7   softmax and epilogue: warps w and w + 4 have the same 32 rows (TMEM lanes), a thread is a row, and each takes
//         half of a block's keys and of O's columns.  They exchange their maxima every stage.
//   8     loads its half of the K blocks (TMA, one box of rows per page and 64 dims).
//   9     loads its half of the V blocks.
//   10    in the pair's first CTA: issues the MMAs of both.  S of stage i + 1 before O of stage i, so that the
//         softmax of a stage runs under the next stage's scores and the last one's product.
//   11    tells the first CTA that a K block has landed in this one.
//   12-15 load the queries (whole tokens by TMA, else row by row), and look through V blocks that not every row sees: a
//         value that is not finite becomes 0 (0 x inf is NaN), and the rows that see it get it in the epilogue.  Then
//         they tell the first CTA.
// Barriers that both CTAs arrive on lie in the first CTA.  Every wait is bounded; a thread that gives up sets the
// abort flags of both CTAs and the error word, all waits then end at once, and both free their TMEM and leave.
#include <float.h>

#include <algorithm>
#include <atomic>

#include "g4a_chunk_pair.cuh"

namespace {

using namespace g4a;
using namespace g4a_chunk;

constexpr int kThreadsC = 512;
constexpr int kSoft = 8, kLoadK = 8, kLoadV = 9, kMma = 10, kTellK = 11, kGuard = 12;
constexpr int kCtaRows = 128;
// Weights are p = 2^(s - m).  A score above m + 15 (f16 ends at 2^16) raises m to 3 below it, so the largest weight is 2^3 at
// least, and f16's rounding of one is off by 2^-11 of it or, below 2^-14, by 2^-25, which is 2^-28 of the largest.  A raise costs
// the pair a stage's time (O has to be at rest to be rescaled), so m does not follow the maximum closely: with m kept 7 below
// the maximum and raised at 2^8 past it, 512 tokens over 131,000 rows took 591 us instead of 447, six ragged chunks of
// heads of 128 dims 213 instead of 190.  With later raises to 1 above the maximum, which leave the most room, both took
// the same time as now, and one row found late left 131,000 rows at 2^-24.2 of it no weight at all.
constexpr float kRaiseC = 15.0f, kBelowC = 3.0f;
constexpr float kUnseenC = -FLT_MAX;  // m of a row that has seen nothing yet (any finite score raises it)
constexpr int kBadTags = 8;

template <int HD>
struct Cc {
  static constexpr int HDV = HD > 256 ? 256 : HD;    // dims of O of a piece
  static constexpr int HALVES = HD / HDV;
  static constexpr int KB_LOG2 = HD > 256 ? 6 : 7;
  static constexpr int KB = 1 << KB_LOG2;            // keys of a block
  static constexpr int NCQ = HD / 64, NCV = HDV / 128;  // 64-dim chunks of Q and K, of this CTA's share of V
  static constexpr int Q_CHUNK = kCtaRows * 128, K_CHUNK = KB / 2 * 128, V_CHUNK = KB * 128;
  static constexpr int Q_BYTES = NCQ * Q_CHUNK, K_BYTES = NCQ * K_CHUNK, V_BYTES = NCV * V_CHUNK;
  static constexpr int NS = HD <= 128 ? 4 : 2;       // K and V blocks in flight
  static constexpr bool OWN_STAGING = HD <= 256;     // (else the epilogue goes through Q's place)
  static constexpr int OFF_Q = 0, OFF_K = OFF_Q + Q_BYTES, OFF_V = OFF_K + NS * K_BYTES, OFF_END = OFF_V + NS * V_BYTES;
  static constexpr int OFF_OUT = OWN_STAGING ? OFF_END : OFF_Q;  // [8 warps][32 rows][64 B]
  static constexpr int OFF_OK = OFF_END + (OWN_STAGING ? kSoft * 2048 : 0);  // [2 NS][4] which rows of a block are there
  static constexpr int OFF_RED = OFF_OK + 2 * NS * 16;                       // [2][2 halves][128] maxima, sums
  static constexpr int OFF_BAD = OFF_RED + 2 * 2 * kCtaRows * 4;             // [kBadTags] piece + 1 with values taken out
  static constexpr int OFF_BAR = OFF_BAD + kBadTags * 4;
  static constexpr int NBARS = 6 * NS + 15;
  static constexpr size_t SMEM = (size_t)OFF_BAR + NBARS * 8 + 16;
  static constexpr uint32_t COL_O = 0, COL_S = HDV;  // S[b] at COL_S + KB b, P[b] in its first half
  static constexpr uint32_t TMEM_COLS = 512;
  static_assert(COL_S + 2 * KB <= TMEM_COLS && SMEM <= 232448, "tile fits");
  // Registers: 512 threads start with 128; the softmax warps hold half a row of scores.
  static constexpr int REGS_SOFT = 160, REGS_REST = 88;
  static_assert(256 * REGS_SOFT + 256 * REGS_REST <= kThreadsC * 128, "register file");
};

struct TcParams {
  ChunkParams c;
  const Plan* plan;
  const Piece* pieces;
  const Cut* cuts;
  float* part;            // [slots] (o [HDV / 4][256][4] | m [256] | l [256])
  int box_k, box_v;       // rows of a box
  int q_tokens;           // tokens of a CTA's queries where they are whole tokens (one box for 64 dims); 0: row by row
};

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A piece as its roles see it.
template <int HD>
struct Work {
  Piece d;
  int kvh, half, base, first, last;  // first and last token of the tile
  __device__ __forceinline__ Work(const ChunkParams& p, const Piece& piece) : d(piece) {
    kvh = d.head / Cc<HD>::HALVES;
    half = d.head - kvh * Cc<HD>::HALVES;
    base = d.L - d.T;
    first = first_token(p, d.tile);
    last = last_token(p, d.T, d.tile);
  }
  __device__ __forceinline__ int stages() const { return d.j1 - d.j0; }
  __device__ __forceinline__ int key0(int j) const { return (j < d.sinks ? j : j + d.skip) << Cc<HD>::KB_LOG2; }
  // whether every row of the tile sees every key of the block at k0 (if it is there)
  __device__ __forceinline__ bool clean(const ChunkParams& p, int k0) const {
    const int end = k0 + Cc<HD>::KB;
    return end <= base + first + 1 && (k0 >= first_in_window(p, base + last) || (uint32_t)end <= p.sinks);
  }
};

// Adds to what this thread has stored for a row (half of its columns) the infinities and NaN of the V values that were taken out of
// the piece's blocks, where the row sees their keys.
template <int HD>
__device__ __noinline__ void add_taken_out(const ChunkParams& p, Work<HD> w, int pos, size_t out_row, float* part, int row, int half) {
  using C = Cc<HD>;
  const int d0 = w.half * C::HDV, from = d0 + half * (C::HDV / 2), d1 = min(p.hd, from + C::HDV / 2);
  for (int j = w.d.j0; j < w.d.j1; j++) {
    const int k0 = w.key0(j);
    if (w.clean(p, k0)) continue;
    for (int key = k0; key < k0 + C::KB && key <= pos; key++) {
      if (!sees(p, pos, key)) continue;
      const long long off = row_offset(p, w.d.b, w.kvh, key);
      if (off < 0) continue;
      for (int d = from; d < d1; d++) {
        const float v = __half2float(p.v[off + d]);
        if (fabsf(v) < INFINITY) continue;
        if (part != nullptr) {
          const int e = d - d0;
          part[((size_t)(e >> 2) * kTileRows + row) * 4 + (e & 3)] += v;
        } else {
          __half* o = p.out + out_row * p.hd + d;
          *o = __float2half_rn(__half2float(*o) + v);
        }
      }
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreadsC, 1)
    chunk_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                    const __grid_constant__ CUtensorMap tmq, const TcParams a) {
  using C = Cc<HD>;
  const ChunkParams& p = a.c;
  extern __shared__ __align__(1024) unsigned char smem[];  // (at 512 dims there is no room to align it by hand)
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicExch(p.err, G4A_DEVERR_TMEM);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_landed = bars;                 // [NS] this CTA's half of a K block
  uint64_t* v_landed = k_landed + C::NS;     // [NS]
  uint64_t* k_ready = v_landed + C::NS;      // [NS] first CTA: both halves
  uint64_t* p_ready = k_ready + C::NS;       // [NS] first CTA: weights (8 warps of each) and V, looked through (4 of each)
  uint64_t* s_done = p_ready + C::NS;        // [NS] scores (commit), and which rows of the block are there (warp 8)
  uint64_t* o_done = s_done + C::NS;         // [NS] a stage's product done (commit)
  uint64_t* q_ready = o_done + C::NS;        // first CTA: queries of both (4 warps of each)
  uint64_t* q_free = q_ready + 1;            // the piece's last scores done (commit)
  uint64_t* o_free = q_free + 1;             // first CTA: epilogue has read O (8 warps of each)
  // [2] the piece's V blocks have been looked through (4 warps of each).  A warp may be through with a piece before
  // another is with the one before it, so they take turns; it is not two ahead, for the scores of the piece between
  // need every warp's word on its queries.
  uint64_t* looked = o_free + 1;
  uint64_t* staged = looked + 2;             // the epilogue is through with the staging place (8 warps)
  uint64_t* swapped = staged + 1;            // [4] two warps have written what they exchange
  uint64_t* all_done = swapped + 4;
  uint64_t* q_landed = all_done + 1;         // this CTA's queries (TMA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cta_rank();
  const uint32_t sbase = smem_u32(smem);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NS; s++) {
      mbar_init(&k_landed[s], 1);
      mbar_init(&v_landed[s], 1);
      mbar_init(&k_ready[s], 2);
      mbar_init(&p_ready[s], 2 * kSoft + 8);
      mbar_init(&s_done[s], 2);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(q_ready, 8);
    mbar_init(q_free, 1);
    mbar_init(o_free, 2 * kSoft);
    mbar_init(&looked[0], 8);
    mbar_init(&looked[1], 8);
    mbar_init(staged, kSoft);
    for (int s = 0; s < 4; s++) mbar_init(&swapped[s], 2);
    mbar_init(all_done, 1);
    mbar_init(q_landed, 1);
    *abort_flag = 0;
    for (int i = 0; i < kBadTags; i++) reinterpret_cast<int*>(smem + C::OFF_BAD)[i] = 0;
    fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmv)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmq)) : "memory");
  }
  __syncwarp();
  if (warp == kMma) {  // one CTA per SM (shared memory), so the allocation never waits
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

  // this pair's pieces
  const int4 mine = a.plan->pair[blockIdx.x >> 1];
  const int begin = mine.x, end = mine.y, step = mine.z;

  if (warp < kSoft) {
    // ------------------------------------------------------------------ softmax, epilogue
    regs_up<C::REGS_SOFT>();
    const int quarter = warp & 3, half = warp >> 2;  // rows; keys [HB half, HB half + HB) of a block
    constexpr int HB = C::KB / 2, HO = C::HDV / 2;   // and columns [HO half, HO half + HO) of O
    const int cta_row = quarter * 32 + lane, row = rank * kCtaRows + cta_row;  // of the CTA, of the tile
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t p_bar = map_to(smem_u32(p_ready), 0), o_bar = map_to(smem_u32(o_free), 0);
    const volatile int* tags = reinterpret_cast<const volatile int*>(smem + C::OFF_BAD);
    float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
    uint32_t g = 0, done = 0, swaps = 0;  // stages, pieces and exchanges so far
    bool ok = true;
    // This thread's value for the other half's thread of the row, and that one's for this.  The places alternate: a
    // warp writes one again only after the exchange between, for which the other had to come after reading it.
    auto swap = [&](float mine) {
      float* at = red + (swaps & 1u) * (2 * kCtaRows) + cta_row;
      at[half * kCtaRows] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(&swapped[quarter]);
      ok = warp_wait_own(&swapped[quarter], swaps & 1u, abort_flag, p.err);
      swaps++;
      return *reinterpret_cast<volatile float*>(at + (half ^ 1) * kCtaRows);
    };
    for (int i = begin; ok && i < end; i += step) {
      const Work<HD> w(p, a.pieces[i]);
      if (w.stages() <= 0) continue;
      const uint32_t gr = (uint32_t)w.d.tile * kTileRows + (uint32_t)row;
      const bool live = gr < (uint32_t)w.d.T * (uint32_t)p.group;
      const int token = live ? (int)(gr / (uint32_t)p.group) : w.d.T - 1;
      const int pos = w.base + token, lo = first_in_window(p, pos);
      float m = kUnseenC, l = 0.f;
      for (int j = w.d.j0; j < w.d.j1; j++, g++) {
        const uint32_t col = lanes + C::COL_S + (g & 1u) * C::KB;
        ok = warp_wait_own(&s_done[g % C::NS], (g / C::NS) & 1u, abort_flag, p.err);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[HB / 32][32];
#pragma unroll
        for (int c = 0; c < HB / 32; c++) tmem_get(col + half * HB + 32u * c, s[c]);
        const uint32_t* there = reinterpret_cast<const uint32_t*>(smem + C::OFF_OK + (g % (2 * C::NS)) * 16) + half * (HB / 32);
        const uint32_t there0 = there[0], there1 = HB > 32 ? there[1] : 0xffffffffu;
        const int k0 = w.key0(j) + half * HB;
        // from the half block's first key: z the last one seen, f the first one of the window, and sinks before n
        const int z = pos - k0, f = lo - k0;
        const int n = (int)max(min((long long)p.sinks - k0, (long long)HB), 0ll);
        const bool plain = __all_sync(0xffffffffu, z >= HB - 1 && (f <= 0 || n >= HB)) && (there0 & there1) == 0xffffffffu &&
                           p.scale_log2 > 0.f;
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < HB / 32; c++) tmem_landed(s[c]);
        float by = p.scale_log2;
        if (!plain) {
          by = 1.f;
#pragma unroll
          for (int c = 0; c < HB / 32; c++) {
            // bits of keys [32 c, 32 c + 32): up to z, and from f on or before n
            const int zc = z - 32 * c, fc = f - 32 * c, nc = n - 32 * c;
            const uint32_t upto = zc >= 31 ? 0xffffffffu : zc < 0 ? 0u : (2u << zc) - 1u;
            const uint32_t from = fc <= 0 ? 0xffffffffu : fc > 31 ? 0u : ~((1u << fc) - 1u);
            const uint32_t sink = nc >= 32 ? 0xffffffffu : nc <= 0 ? 0u : (1u << nc) - 1u;
            const uint32_t bits = upto & (from | sink) & (c == 0 ? there0 : there1);
#pragma unroll
            for (int e = 0; e < 32; e++)
              s[c][e] = (bits >> e) & 1u ? __float_as_uint(__uint_as_float(s[c][e]) * p.scale_log2) : 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < HB / 32; c++)
#pragma unroll
          for (int e = 0; e < 32; e++) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(s[c][e]));
        const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * by;
        const float top = fmaxf(mine, swap(mine));
        if (!ok) break;
        const bool raise = top > m + kRaiseC;
        if (__any_sync(0xffffffffu, raise)) {  // (both halves agree)
          const float m_new = raise ? top - kBelowC : m;
          const float fall = raise ? (m == kUnseenC ? 0.f : fast_exp2(m - m_new)) : 1.f;
          l *= fall;
          m = m_new;
          if (j > w.d.j0) {
            // O holds the stages up to j - 1, whose product is the last one issued before this stage's
            ok = warp_wait_own(&o_done[(g - 1) % C::NS], ((g - 1) / C::NS) & 1u, abort_flag, p.err);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = half * HO; c < half * HO + HO; c += 32) {
              uint32_t o[32];
              tmem_ld32(lanes + C::COL_O + c, o);
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fall);
              tmem_st32(lanes + C::COL_O + c, o);
            }
          }
        }
        const uint64_t by2 = f32x2(by, by), up2 = f32x2(-m, -m);
        uint64_t sum[2] = {0, 0};
        uint32_t pw[HB / 2];
#pragma unroll
        for (int e = 0; e < HB / 2; e++) {
          const uint64_t x = f32x2(__uint_as_float(s[e >> 4][(2 * e) & 31]), __uint_as_float(s[e >> 4][(2 * e + 1) & 31]));
          const float2 y = f32x2_parts(fma_f32x2(x, by2, up2));
          const float w0 = fast_exp2(y.x), w1 = fast_exp2(y.y);
          sum[e & 1] = add_f32x2(sum[e & 1], f32x2(w0, w1));
          pw[e] = half2_bits(w0, w1);
        }
        // (where the other half's scores were: it has read them, or it would not have come to the exchange)
        if constexpr (HB == 64) tmem_st32(col + half * 32u, pw);
        else tmem_st16(col + half * 16u, pw);
        const float2 total = f32x2_parts(add_f32x2(sum[0], sum[1]));
        l += total.x + total.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(p_bar + (g % C::NS) * 8u);
      }
      if (!ok) break;
      // ---- epilogue
      const float other = swap(l);
      if (!ok) break;
      l = half == 0 ? l + other : other + l;
      ok = warp_wait_own(&o_done[(g - 1) % C::NS], ((g - 1) / C::NS) & 1u, abort_flag, p.err);
      if (!ok) break;
      ok = __all_sync(0xffffffffu, wait_pair(&looked[done & 1u], (done >> 1) & 1u, abort_flag, p.err));
      if (!ok) break;
      const bool bad = tags[done % kBadTags] == (int)done + 1;
      tc_fence_after();
      const size_t out_row = live ? (size_t)(w.d.row0 + token) * p.nqh + (size_t)(w.kvh * p.group) + (gr - (uint32_t)token * (uint32_t)p.group) : 0;
      const unsigned lives = __ballot_sync(0xffffffffu, live);  // (the first ones)
      float* part = w.d.slot < 0 ? nullptr : a.part + (size_t)w.d.slot * kTileRows * (C::HDV + 2);
      if (part != nullptr) {
#pragma unroll 1
        for (int c = half * HO; c < half * HO + HO; c += 32) {
          uint32_t o[32];
          tmem_ld32(lanes + C::COL_O + c, o);
          if (live)
#pragma unroll
            for (int e = 0; e < 8; e++)
              *reinterpret_cast<uint4*>(part + ((size_t)(c / 4 + e) * kTileRows + row) * 4) =
                  make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        if (live && half == 0) {
          part[(size_t)C::HDV * kTileRows + row] = m;
          part[(size_t)(C::HDV + 1) * kTileRows + row] = l;
        }
      } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        unsigned char* stage = smem + C::OFF_OUT + warp * 2048;
#pragma unroll 1
        for (int c = half * HO; c < half * HO + HO; c += 32) {  // 32 columns of the warp's 32 rows through shared memory
          uint32_t o[32];
          tmem_ld32(lanes + C::COL_O + c, o);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint4 x;
            x.x = half2_bits(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
            x.y = half2_bits(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
            x.z = half2_bits(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
            x.w = half2_bits(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) = x;
          }
          __syncwarp();
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 8) {
            const int r = r0 + (lane >> 2), e = lane & 3, d = w.half * C::HDV + c + e * 8;
            const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 64 + ((e ^ ((r >> 1) & 3)) << 4));
            const size_t at = __shfl_sync(0xffffffffu, out_row, r);
            if (((lives >> r) & 1u) && d < p.hd) *reinterpret_cast<uint4*>(p.out + at * p.hd + d) = x;
          }
          __syncwarp();
        }
        if (p.lse != nullptr && live && w.half == 0 && half == 0)
          p.lse[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2C;
      }
      if (bad && live) add_taken_out<HD>(p, w, pos, out_row, part, row, half);
      tc_fence_before();
      // the next queries are copied by TMA to where this output has been
      if (!C::OWN_STAGING) fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (!C::OWN_STAGING) mbar_arrive(staged);  // (before o_free, without which no warp gets through another piece)
        arrive_at(o_bar);
      }
      done++;
    }
  } else {
    regs_down<C::REGS_REST>();
    if (warp == kLoadK || warp == kLoadV) {
      // ---------------------------------------------------------------- loads
      const bool kside = warp == kLoadK;
      uint64_t* landed = kside ? k_landed : v_landed;
      uint64_t* free_bar = kside ? s_done : o_done;  // (of stage g - NS)
      const CUtensorMap* map = kside ? &tmk : &tmv;
      const int box = kside ? a.box_k : a.box_v, rows = kside ? C::KB / 2 : C::KB, chunks = kside ? C::NCQ : C::NCV;
      const int chunk_bytes = kside ? C::K_CHUNK : C::V_CHUNK, bytes = kside ? C::K_BYTES : C::V_BYTES;
      const int boxes = rows / box, ops = boxes * chunks;
      const long long cap = (long long)p.max_pages * p.page_size;
      uint32_t g = 0;
      bool ok = true;
      for (int i = begin; ok && i < end; i += step) {
        const Work<HD> w(p, a.pieces[i]);
        const int* table = p.page_table + (size_t)w.d.b * p.max_pages;
        for (int j = w.d.j0; j < w.d.j1; j++, g++) {
          const uint32_t s = g % C::NS;
          if (g >= (uint32_t)C::NS) {
            ok = warp_wait_own(&free_bar[s], (g / C::NS - 1) & 1u, abort_flag, p.err);
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&landed[s], (uint32_t)bytes);
          __syncwarp();
          const int k0 = w.key0(j);
          const uint32_t dst = sbase + (kside ? C::OFF_K : C::OFF_V) + s * bytes;
          for (int o = lane; o < ops; o += 32) {
            const int r = o / chunks, c = o - r * chunks;
            const int key = k0 + (kside ? rank * (C::KB / 2) : 0) + r * box;
            int page = p.num_pages, row = 0;  // a page that is not there: zeros
            if (key < w.d.L) {
              const int t = key / p.page_size, id = table[t];
              row = key - t * p.page_size;
              if (id >= 0 && id < p.num_pages) page = id;
            }
            const int x = kside ? 64 * c : w.half * C::HDV + rank * (C::HDV / 2) + 64 * c;
            load_box(dst + c * chunk_bytes + r * box * 128, map, x, w.kvh, row, page, &landed[s]);
          }
          if (kside) {
            // which of the block's rows are there
            bool gone = false;
            for (int o = lane; o < 2 * boxes; o += 32) {
              const int key = k0 + o * box;
              if (key >= w.d.L) continue;
              const int id = table[key / p.page_size];
              gone |= id < 0 || id >= p.num_pages;
            }
            // (places for twice the ring: this stage's may be written while the softmax is still at stage g - NS)
            uint32_t* to = reinterpret_cast<uint32_t*>(smem + C::OFF_OK + (g % (2 * C::NS)) * 16);
            if (!__any_sync(0xffffffffu, gone)) {
              if (lane < 4) to[lane] = 0xffffffffu;
            } else {
              if (lane == 0) atomicExch(p.err, G4A_DEVERR_PAGE);
#pragma unroll 1
              for (int c = 0; c < 4; c++) {
                const int key = k0 + 32 * c + lane;
                bool here = false;
                if (c < C::KB / 32 && key < w.d.L && key < cap) {
                  const int id = table[key / p.page_size];
                  here = id >= 0 && id < p.num_pages;
                }
                const uint32_t bits = __ballot_sync(0xffffffffu, here);
                if (lane == 0) to[c] = bits;
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_done[s]);
          }
        }
      }
      // loads still in flight land before the CTA leaves (bounded)
      for (uint32_t k = g > (uint32_t)C::NS ? g - C::NS : 0; k < g; k++)
        (void)mbar_wait_bounded(&landed[k % C::NS], (k / C::NS) & 1u, p.err, G4A_DEVERR_WAIT_FULL);
    } else if (warp == kTellK) {
      // ---------------------------------------------------------------- K blocks landed
      if (lane == 0) {
        uint32_t g = 0;
        bool ok = true;
        for (int i = begin; ok && i < end; i += step) {
          const int n = a.pieces[i].j1 - a.pieces[i].j0;
          for (int j = 0; j < n; j++, g++) {
            ok = wait_own(&k_landed[g % C::NS], (g / C::NS) & 1u, abort_flag, p.err);
            if (!ok) break;
            arrive_at(map_to(smem_u32(&k_ready[g % C::NS]), 0));
          }
        }
      }
    } else if (warp == kMma) {
      // ---------------------------------------------------------------- MMAs
      if (rank == 0) {
        const uint32_t on = elect_one();
        constexpr uint32_t idesc_s = pair_idesc(C::KB, false), idesc_o = pair_idesc(C::HDV, true);
        const uint64_t dq = sw128_desc(sbase + C::OFF_Q, 16, 1024);
        const uint64_t dk0 = sw128_desc(sbase + C::OFF_K, 16, 1024);
        // V as the MN-major B operand: 64 dims per 128-byte row, chunks of dims V_CHUNK apart, 8-key groups 1024
        const uint64_t dv0 = sw128_desc(sbase + C::OFF_V, (uint32_t)C::V_CHUNK, 1024);
        uint32_t g = 0, done = 0;
        bool ok = true;
        auto scores = [&](uint32_t k) {
          if (!warp_wait_own(&k_ready[k % C::NS], (k / C::NS) & 1u, abort_flag, p.err)) return false;
          tc_fence_after();
          const uint64_t dk = dk0 + (uint64_t)(((k % C::NS) * C::K_BYTES) >> 4);
          const uint32_t d = tmem + C::COL_S + (k & 1u) * C::KB;
#pragma unroll
          for (int kk = 0; kk < HD / 16; kk++) {
            const uint64_t off = (uint64_t)(((kk & 3) * 32) >> 4);
            mma2_ss(on, d, dq + (uint64_t)(((kk >> 2) * C::Q_CHUNK) >> 4) + off, dk + (uint64_t)(((kk >> 2) * C::K_CHUNK) >> 4) + off,
                    idesc_s, kk > 0 ? 1u : 0u);
          }
          commit2(on, &s_done[k % C::NS]);
          return true;
        };
        for (int i = begin; ok && i < end; i += step) {
          const Work<HD> w(p, a.pieces[i]);
          const int n = w.stages();
          if (n <= 0) continue;
          ok = warp_wait_pair(q_ready, done & 1u, abort_flag, p.err) && scores(g);
          if (ok && n == 1) commit2(on, q_free);
          for (int j = 0; ok && j < n; j++, g++) {
            if (j + 1 < n) {
              ok = scores(g + 1);
              if (!ok) break;
              if (j + 2 == n) commit2(on, q_free);
            }
            // (the epilogue of the piece before has read O)
            if (j == 0 && done > 0) ok = warp_wait_own(o_free, (done - 1) & 1u, abort_flag, p.err);
            // (where V was looked through, there are stores of the other CTA to be seen)
            ok = ok && (w.clean(p, w.key0(w.d.j0 + j)) ? warp_wait_own(&p_ready[g % C::NS], (g / C::NS) & 1u, abort_flag, p.err)
                                                       : warp_wait_pair(&p_ready[g % C::NS], (g / C::NS) & 1u, abort_flag, p.err));
            if (!ok) break;
            tc_fence_after();
            const uint64_t dv = dv0 + (uint64_t)(((g % C::NS) * C::V_BYTES) >> 4);
            const uint32_t pa = tmem + C::COL_S + (g & 1u) * C::KB;
#pragma unroll
            for (int kk = 0; kk < C::KB / 16; kk++)
              mma2_ts(on, tmem + C::COL_O, pa + (uint32_t)(8 * kk), dv + (uint64_t)((kk * 2048) >> 4), idesc_o,
                      j > 0 || kk > 0 ? 1u : 0u);
            commit2(on, &o_done[g % C::NS]);
          }
          done++;
        }
        // no MMA may still be running when TMEM is freed, also after an abort
        commit2(on, all_done);
        (void)mbar_wait_bounded(all_done, 0, p.err, G4A_DEVERR_WAIT_MMA);
      }
    } else {
      // ---------------------------------------------------------------- queries, a look through V
      const int gw = warp - kGuard;
      const uint32_t q_bar = map_to(smem_u32(q_ready), 0);
      const uint32_t tags = sbase + C::OFF_BAD;
      uint32_t g = 0, done = 0;
      bool ok = true;
      for (int i = begin; ok && i < end; i += step) {
        const Work<HD> w(p, a.pieces[i]);
        if (w.stages() <= 0) continue;
        if (done > 0) {
          ok = warp_wait_own(q_free, (done - 1) & 1u, abort_flag, p.err);
          if (ok && !C::OWN_STAGING) ok = warp_wait_own(staged, (done - 1) & 1u, abort_flag, p.err);
          if (!ok) break;
        }
        const uint32_t gr0 = (uint32_t)w.d.tile * kTileRows + (uint32_t)(rank * kCtaRows + gw);
        if (a.q_tokens > 0) {
          // (rows past the sequence's last token are another's, or zeros: what comes of them is not stored)
          if (gw == 0) {
            if (lane == 0) mbar_arrive_expect_tx(q_landed, (uint32_t)C::Q_BYTES);
            __syncwarp();
            const long long token = (long long)w.d.row0 + (long long)(w.d.tile * 2 + rank) * a.q_tokens;
            if (lane < C::NCQ)
              load_box(sbase + C::OFF_Q + lane * C::Q_CHUNK, &tmq, 64 * lane, 0, w.kvh, (int)min(token, (long long)p.tokens), q_landed);
            ok = mbar_wait_bounded(q_landed, done & 1u, p.err, G4A_DEVERR_WAIT_FULL);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          if (lane == 0) arrive_at(q_bar);
        } else {
          const uint32_t rows = (uint32_t)w.d.T * (uint32_t)p.group, group = (uint32_t)p.group;
          const uint32_t up = 4u / group, over = 4u - up * group;  // four rows on: tokens, heads
          uint32_t token = gr0 / group, head = gr0 - token * group;
#pragma unroll 4
          for (int r = gw; r < kCtaRows; r += 4) {
            const bool live = gr0 + (uint32_t)(r - gw) < rows;
            const __half* from = p.q + ((size_t)(w.d.row0 + (int)token) * p.nqh + (size_t)(w.kvh * p.group) + head) * p.hd;
            const uint32_t to = sbase + C::OFF_Q + r * 128;
#pragma unroll
            for (int e = lane; e < HD / 8; e += 32) {
              const bool in = live && e * 8 < p.hd;
              cp16(to + (e >> 3) * C::Q_CHUNK + (((e & 7) ^ (r & 7)) << 4), in ? from + e * 8 : p.q, in);
            }
            token += up;
            head += over;
            if (head >= group) head -= group, token++;
          }
          cp_wait_all();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) publish_at(q_bar);
        }
        const int lo = first_in_window(p, w.base + w.first), hi = w.base + w.last + 1;
        bool found = false;
        for (int j = w.d.j0; j < w.d.j1; j++, g++) {
          const uint32_t s = g % C::NS;
          ok = warp_wait_own(&v_landed[s], (g / C::NS) & 1u, abort_flag, p.err);
          if (!ok) break;
          const int k0 = w.key0(j);
          const bool clean = w.clean(p, k0);
          bool changed = false;
          if (!clean) {
            unsigned char* v = smem + C::OFF_V + s * C::V_BYTES;
#pragma unroll 4
            for (int e = gw * 32 + lane; e < C::V_BYTES / 16; e += 128) {
              uint4 x = *reinterpret_cast<const uint4*>(v + e * 16);
              // an exponent of all ones and one more carry into a half's top bit
              constexpr uint32_t kExp = 0x7c007c00u, kOne = 0x04000400u, kTop = 0x80008000u;
              if ((((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) | ((x.w & kExp) + kOne)) & kTop) {
                auto finite = [](uint32_t w) {
                  const uint32_t top = ((w & kExp) + kOne) & kTop;
                  return w & ~((top >> 15) * 0xffffu);
                };
                *reinterpret_cast<uint4*>(v + e * 16) = make_uint4(finite(x.x), finite(x.y), finite(x.z), finite(x.w));
                changed = true;
                const int key = k0 + (e >> 3) % C::KB;  // 8 pieces of 16 bytes to a row, KB rows to a chunk
                found |= key < hi && (key >= lo || (uint32_t)key < p.sinks);
              }
            }
            if (changed) fence_proxy_async_smem();
          }
          changed = __any_sync(0xffffffffu, changed);
          if (lane == 0) {
            const uint32_t to = map_to(smem_u32(&p_ready[s]), 0);
            if (changed) publish_at(to);
            else arrive_at(to);
          }
        }
        if (!ok) break;
        const bool any = __any_sync(0xffffffffu, found);
        // (a CTA has half of the dims and half of the rows, so both have to know)
#pragma unroll
        for (uint32_t c = 0; c < 2; c++) {
          if (found)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to(tags + (done % kBadTags) * 4, c)), "r"(done + 1) : "memory");
          __syncwarp();
          if (lane == 0) {
            const uint32_t to = map_to(smem_u32(&looked[done & 1u]), c);
            if (any) publish_at(to);
            else arrive_at(to);
          }
        }
        done++;
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
  if (warp == kMma)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
}

// Joins the parts of the tiles that several pieces share.  A task is 8 rows x 64 dims of a cut tile for one warp, whose
// lane has four float4 of a row; where a tile has many parts, 2, 4 or 8 warps share them and meet in shared memory.
// All of a warp's loads of up to four parts are under way together: the kernel is one round of latency and what the
// parts take from the L2 (32 MB of parts: 85 us with a warp for 16 dims of a row's every eighth part, 11 us so).
constexpr int kJoinThreads = 256, kJoinX = 32, kJoinY = 37;
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) chunk_join_kernel(const TcParams a) {
  using C = Cc<HD>;
  const ChunkParams& p = a.c;
  __shared__ float4 so[8][4][32];
  __shared__ float sm[8][8], sl[8][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r8 = lane >> 2, c4 = lane & 3;
  pdl_wait_primary();
  pdl_launch_dependents();
  constexpr int kBlocks = C::HDV / 64;
  const int cuts = a.plan->cuts;
  for (int c = (int)blockIdx.y; c < cuts; c += (int)gridDim.y) {
    const Cut cut = a.cuts[c];
    const int share_log2 = cut.parts <= 4 ? 0 : cut.parts <= 8 ? 1 : cut.parts <= 16 ? 2 : 3;  // warps of a task
    const int live = (int)min((uint32_t)cut.T * (uint32_t)p.group - (uint32_t)cut.tile * kTileRows, (uint32_t)kTileRows);
    const int tasks = (live + 7) / 8 * kBlocks, per = 8 >> share_log2;
    for (int t0 = (int)blockIdx.x * per; t0 < tasks; t0 += (int)gridDim.x * per) {
      const int task = t0 + (warp >> share_log2), part0 = warp & ((1 << share_log2) - 1), stride = 1 << share_log2;
      const int block = task % kBlocks, row = task / kBlocks * 8 + r8;
      const bool in = task < tasks && row < live;
      float m = -INFINITY, l = 0.f;
      float4 o[4];
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in) {
        constexpr int kFly = 4;
        for (int i0 = part0; i0 < cut.parts; i0 += stride * kFly) {
          float mi[kFly], li[kFly];
          float4 x[kFly][4];
#pragma unroll
          for (int f = 0; f < kFly; f++) {
            const int i = i0 + stride * f;
            mi[f] = -INFINITY, li[f] = 0.f;
            const float* part = a.part + (size_t)cut.slot_of(i) * kTileRows * (C::HDV + 2);
            if (i < cut.parts) {
              mi[f] = __ldcg(part + (size_t)C::HDV * kTileRows + row);
              li[f] = __ldcg(part + (size_t)(C::HDV + 1) * kTileRows + row);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
              x[f][k] = i < cut.parts ? __ldcg(reinterpret_cast<const float4*>(part) + (size_t)(block * 16 + 4 * k + c4) * kTileRows + row)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          float mn = m;
#pragma unroll
          for (int f = 0; f < kFly; f++) mn = fmaxf(mn, mi[f]);
          const float wo = m == mn ? 1.f : fast_exp2(m - mn);
          m = mn;
          l *= wo;
#pragma unroll
          for (int k = 0; k < 4; k++) o[k].x *= wo, o[k].y *= wo, o[k].z *= wo, o[k].w *= wo;
#pragma unroll
          for (int f = 0; f < kFly; f++) {
            // a part that saw nothing has weight 0 or sums of 0
            const float wf = mi[f] == mn ? 1.f : fast_exp2(mi[f] - mn);
            l = fmaf(wf, li[f], l);
#pragma unroll
            for (int k = 0; k < 4; k++) {
              o[k].x = fmaf(wf, x[f][k].x, o[k].x);
              o[k].y = fmaf(wf, x[f][k].y, o[k].y);
              o[k].z = fmaf(wf, x[f][k].z, o[k].z);
              o[k].w = fmaf(wf, x[f][k].w, o[k].w);
            }
          }
        }
      }
      if (share_log2 > 0) {  // (the same for the whole CTA)
        if (c4 == 0) sm[warp][r8] = m, sl[warp][r8] = l;
#pragma unroll
        for (int k = 0; k < 4; k++) so[warp][k][lane] = o[k];
        __syncthreads();
        if (in && part0 == 0) {
          float mx = m;
          for (int i = 1; i < stride; i++) mx = fmaxf(mx, sm[warp + i][r8]);
          l = 0.f;
#pragma unroll
          for (int k = 0; k < 4; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int i = 0; i < stride; i++) {
            const float wf = sm[warp + i][r8] == mx ? 1.f : fast_exp2(sm[warp + i][r8] - mx);
            l = fmaf(wf, sl[warp + i][r8], l);
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float4 x = so[warp + i][k][lane];
              o[k].x = fmaf(wf, x.x, o[k].x);
              o[k].y = fmaf(wf, x.y, o[k].y);
              o[k].z = fmaf(wf, x.z, o[k].z);
              o[k].w = fmaf(wf, x.w, o[k].w);
            }
          }
          m = mx;
        }
      }
      if (in && part0 == 0) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int kvh = cut.head / C::HALVES, half = cut.head - kvh * C::HALVES;
        const uint32_t gr = (uint32_t)cut.tile * kTileRows + (uint32_t)row, token = gr / (uint32_t)p.group;
        const size_t to = (size_t)(cut.row0 + (int)token) * p.nqh + (size_t)(kvh * p.group) + (gr - token * (uint32_t)p.group);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int d = half * C::HDV + block * 64 + k * 16 + c4 * 4;
          if (d < p.hd)
            *reinterpret_cast<uint2*>(p.out + to * p.hd + d) =
                make_uint2(half2_bits(o[k].x * inv, o[k].y * inv), half2_bits(o[k].z * inv, o[k].w * inv));
        }
        if (p.lse != nullptr && block == 0 && half == 0 && c4 == 0) p.lse[to] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2C;
      }
      if (share_log2 > 0) __syncthreads();
    }
  }
}

template <int HD>
g4a_status launch_chunk(g4a_ctx* ctx, const ChunkParams& p) {
  using C = Cc<HD>;
  const char* fn = "g4a_chunk_attn_paged";
  static std::atomic<bool> ready[64];
  if (ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(chunk_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(chunk_tc_kernel)");
    if (ctx->device < 64) ready[ctx->device].store(true, std::memory_order_release);
  }
  TcParams a = {};
  a.c = p;
  // a box of rows lies in one page: the largest power of two that divides the page
  const int unit = p.page_size & -p.page_size;
  a.box_k = std::min(unit, C::KB / 2);
  a.box_v = std::min(unit, C::KB);
  CUtensorMap mk, mv, mq;
  if (g4a_status s = g4a_page_map(fn, ctx, &mk, p, p.k, a.box_k)) return s;
  if (g4a_status s = g4a_page_map(fn, ctx, &mv, p, p.v, a.box_v)) return s;
  a.q_tokens = kCtaRows % p.group == 0 ? kCtaRows / p.group : 0;
  if (g4a_status s = g4a_query_map(fn, ctx, &mq, p, a.q_tokens > 0 ? p.group : 1, std::max(a.q_tokens, 1))) return s;
  const int pairs = std::min(ctx->num_sms / 2, kMaxPairs);
  const long long entries = (long long)p.tokens * p.group / kTileRows + std::min(p.batch, p.tokens);
  const long long items = entries * p.nkh * C::HALVES;
  if (items > (1 << 24)) return g4a_fail(G4A_EINVAL, "%s: num_tokens * num_q_heads too large", fn);
  const long long slots = 4ll * pairs, pieces = items + slots;  // (runs: an item's piece for pair w lies at item + w)
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  const size_t n_part = up((size_t)slots * kTileRows * (C::HDV + 2) * sizeof(float)), n_plan = up(sizeof(Plan));
  const size_t n_piece = up((size_t)pieces * sizeof(Piece)), n_cut = up((size_t)items * sizeof(Cut));
  const size_t n_seq = up((size_t)(p.batch + 1) * sizeof(int4)), n_entry = up((size_t)entries * sizeof(long long));
  if (g4a_status s = g4a_ensure_workspace(ctx, n_part + n_plan + n_piece + n_cut + n_seq + n_entry)) return s;
  char* ws = static_cast<char*>(ctx->workspace);
  PlanParams q = {};
  q.c = p;
  q.pairs = pairs;
  q.halves = C::HALVES;
  q.kb_log2 = C::KB_LOG2;
  q.max_slots = (int)slots;
  q.max_entries = entries;
  q.stage_bytes = 2.f * (C::K_BYTES + C::V_BYTES);
  q.part_bytes = (float)(kTileRows * C::HDV * sizeof(float));
  q.stage_ns = C::KB * (HD + C::HDV) * (1.f / 55.f);
  a.part = reinterpret_cast<float*>(ws);
  q.plan = reinterpret_cast<Plan*>(ws += n_part);
  q.pieces = reinterpret_cast<Piece*>(ws += n_plan);
  q.cuts = reinterpret_cast<Cut*>(ws += n_piece);
  q.seqs = reinterpret_cast<int4*>(ws += n_cut);
  q.entries = reinterpret_cast<long long*>(ws += n_seq);
  a.plan = q.plan;
  a.pieces = q.pieces;
  a.cuts = q.cuts;
  g4a_prof_scope ps(ctx, G4A_PROF_CHUNK_ATTN);
  cudaError_t e = g4a_chunk_plan_launch(ctx, q, false, entries);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_plan_kernel");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kThreadsC);
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
  e = cudaLaunchKernelEx(&cfg, chunk_tc_kernel<HD>, mk, mv, mq, a);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_tc_kernel");
  e = g4a_launch(chunk_join_kernel<HD>, dim3(kJoinX, kJoinY), dim3(kJoinThreads), 0, ctx->stream, true, a);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_join_kernel");
  return G4A_OK;
}

}  // namespace

g4a_status g4a_chunk_tc_launch(g4a_ctx* ctx, const ChunkParams& p) {
  if (p.hd > 256) return launch_chunk<512>(ctx, p);
  if (p.hd > 128) return launch_chunk<256>(ctx, p);
  return launch_chunk<128>(ctx, p);
}
