// The tensor-core kernel of g4a_tree_attn_paged (tcgen05 / TMEM), and why it is turned round.
//
// A tcgen05 MMA computes 128 x N with N from 16 up.  Here the plentiful dimension is the keys and
// the head dims, and the query rows are few (8 to a few hundred), so the products are transposed:
//   S^T [128 keys x N] = K [128 x hd] Q^T          A = K tile, B = the tile's queries
//   O^T [hd x N]      += V^T [hd x 128] P^T        A = V tile (MN-major), B = P (MN-major)
// The 128 side is always full, the work grows with the rows that exist, and at head_dim 512 the
// accumulator of 64 rows takes 4 x 64 TMEM columns where [rows x 512] would take all 512.  TMEM
// lane = key (scores) or head dim (output), column = query row.
//   f16 queries: a column is a query row (32 or 64 of them; of 64 columns the upper half idles at 32).
//   f32 queries: N columns are N / 2 rows, first their high, then their low f16 terms (of Q and of
//   P), so one MMA of N columns multiplies both; a thread adds a row's two columns itself.
//
// Bound.  A stage is 128 keys.  At head_dim 512 its 256 KB take 11,000 cycles at an SM's share of the HBM
// rate (23 B / cycle).  Shared memory, 128 B / cycle, is the next limit: an MMA of M 128, N 64, K 16 reads 6
// KB (48 cycles; 8 KB and 64 at N 128), so a stage of 64 columns moves 393 KB of operands and 256 KB of
// copies, 5,100 cycles.  So one tile per kv head is bound by HBM and many by shared memory:
//   8 tokens x 8 heads of 512 dims over 131,000 keys, f16: 69 us, 3.9 TB/s (0.59 of the measured copy)
//   48 tokens, six tiles: 183 us, 564 TFLOP/s, 6,700 cycles a stage (201 us at the clock that the power limit
//   leaves after some 10 ms of such calls one after another, 1,760 MHz)
//   the same with f32 queries, 32 rows to a tile: 81 us and 336 us
// Below 512 dims the softmax warps' serial chain, S -> registers -> vote -> exp2 -> P, is longer than the
// products: 3,600 cycles at 32 rows a warp (8 tiles of 256 dims over 32k keys: 4,900 a stage, 60 us), 1,950 at 16
// (32 chains of up to 7 tokens x 3 heads of 128 dims, 3,000 keys: 2,830 a stage, which is the HBM share; 44 us).
// Short calls are bound by latency: 14 us at one stage (f16), of which the start up to the first keys' arrival
// is 5 us (3 of them to find this CTA's stages, in cold code), a stage 3, the epilogue 1 to 2, the join 3 to 4.
//
// Shared memory: Q [64-dim chunk][N][128 B], P [64-column chunk][128 keys][128 B], and a ring of
// 32 KB units, each 128 keys x 128 dims of K or V as two [128 keys][128 B] chunks, all with the
// 128-byte swizzle (16-byte piece k of row r at k ^ (r & 7)).
// Warps (16):
//   0-7    softmax: warp w has TMEM lanes 32 (w % 4) .. + 31 (keys) and the rows of half w / 4.
//          A thread holds one key's scores for its rows.  The running maximum of a row is raised
//          only when a score passes it by 2^8 (p = 2^(s - m + 7) <= 2^15 stays in f16): whether
//          any does is one vote of a half's four warps per stage; finding the maxima (a transposing
//          reduction over the lanes and the four warps) and rescaling O in TMEM happens only then.
//          (16 warps with half the rows each had 80 registers and no gain at 64 rows: 212 us for
//          the six tiles above.)
//   8-11   loads: row addresses through the page table (any page size), cp.async into the ring
//          with zero fill for rows that are not there, and the tile's queries (f32 queries as the
//          terms that a small kernel before this one has split them into).
//   12     issues the MMAs: S of stage i, then O of stage i - 1, so the softmax of a stage runs under
//          the next stage's score product.
//   13-15  hand landed units over to the MMA warp (proxy fence), V values checked on the way.
// Every wait is bounded; a thread that gives up sets the abort flag and the error word, all waits
// then end at once, and the CTA frees its TMEM and leaves.
#include <float.h>

#include <algorithm>
#include <atomic>

#include "g4a_tcgen05.cuh"
#include "g4a_tree.cuh"

namespace {

using namespace g4a;
using namespace g4a_tree;

constexpr int kKeysT = 1 << kStageLog2;
constexpr int kMaxGrid = 256;        // (the join looks at one cut per thread)
constexpr int kSoftWarps = 8;        // two for each lane quarter: the rows in two shares
constexpr int kLoadWarp = kSoftWarps, kMmaWarp = kLoadWarp + 4;
constexpr int kThreadsTc = (kMmaWarp + 4) * 32;  // softmax, loading, MMA and handing over
constexpr int kShares = kSoftWarps / 4;
constexpr int kUnit = 32768;         // 128 keys x 128 dims f16
constexpr float kPUp = 7.0f;         // p = 2^(s - m + 7)
constexpr float kRaise = 8.0f;       // a score this far above m raises it
constexpr float kUnseen = -FLT_MAX;  // m of a row that has seen nothing yet (any finite score raises it)

template <int HD, int N, bool F32, int R>
struct Tc {
  static constexpr int MB = HD / 128;                 // 128-dim blocks = ring units of a K or V tile
  static constexpr int ROWS = R;                      // query rows of a tile
  static constexpr int W = ROWS / kShares;            // rows of a softmax warp (its share)
  // Registers: 512 threads start with 128 each (65,536); the softmax warps, which hold a block of
  // scores and the row sums, take some from the others.  (Spills are dear here: shared memory leaves
  // the L1 almost nothing, so local memory is in the L2.  The two f32 instances of 64 rows store 36 and 40
  // bytes a thread, the others none.)
  static constexpr int REGS_SOFT = 160, REGS_LOAD = 112, REGS_MMA = 80;
  static_assert(kSoftWarps * 32 * REGS_SOFT + 128 * REGS_LOAD + 128 * REGS_MMA <= kThreadsTc * 128, "register file");
  static constexpr int Q_BYTES = N * HD * 2;
  static constexpr int P_BYTES = kKeysT * N * 2;
  static constexpr int FIT2 = (216 * 1024 - 2 * Q_BYTES - P_BYTES) / kUnit;
  static constexpr int NQ = FIT2 >= 4 ? 2 : 1;        // query buffers
  static constexpr int FIT = (216 * 1024 - NQ * Q_BYTES - P_BYTES) / kUnit;
  static constexpr int UNITS = FIT > 5 ? 5 : FIT;
  static constexpr int OFF_P = NQ * Q_BYTES;
  static constexpr int OFF_RING = OFF_P + P_BYTES;
  static constexpr int OFF_SEES = OFF_RING + UNITS * kUnit;   // [4][ROWS] Sees
  static constexpr int OFF_SCALE = OFF_SEES + 4 * ROWS * 16;  // [4][ROWS]
  static constexpr int OFF_U = OFF_SCALE + 4 * ROWS * 4;      // [softmax warps][W] m - 7 of its rows
  static constexpr int OFF_F = OFF_U + kSoftWarps * W * 4;    // [softmax warps][W] rescale factors
  static constexpr int OFF_MAX = OFF_F + kSoftWarps * W * 4;  // [shares][4 quarters][W]
  static constexpr int OFF_SUM = OFF_MAX + kSoftWarps * W * 4; // [shares][4 quarters][W]
  static constexpr int OFF_OK = OFF_SUM + kSoftWarps * W * 4; // [8 stages][4] which rows are there
  static constexpr int OFF_BAD = OFF_OK + 128;                // [8] tile + 1 that had a V value that is not finite
  static constexpr int OFF_VOTE = OFF_BAD + 32;               // [shares][2][4 quarters]
  static constexpr int OFF_INFO = OFF_VOTE + kShares * 32;               // [4] Walk of a piece's begin
  static constexpr int OFF_BAR = OFF_INFO + 4 * 64;
  static constexpr int NBARS = 3 * UNITS + 8 + 2 + 8 + 2 + 8 + 3 + kShares;
  static constexpr int OFF_END = OFF_BAR + NBARS * 8;
  static constexpr size_t SMEM = 1024 + OFF_END + 16;
  static constexpr uint32_t COL_O = 0, COL_S = MB * N;
  static constexpr uint32_t TMEM_COLS = COL_S + 2 * N <= 256 ? 256u : 512u;
  // (the queries are handed over after a stage's K units, so the ring has to hold those: UNITS >= MB)
  static_assert(COL_S + 2 * N <= 512 && UNITS >= 3 && UNITS >= MB && SMEM <= 232448, "tile fits");
};

template <int R>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrives on `bar` (one of its expected count) when this thread's copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Sets infinite and NaN halves of a pair to 0; whether there was one.
__device__ __forceinline__ bool clear_non_finite(uint32_t& w) {
  uint32_t keep = 0xffffffffu;
  if ((w & 0x7c00u) == 0x7c00u) keep &= 0xffff0000u;
  if ((w & 0x7c000000u) == 0x7c000000u) keep &= 0x0000ffffu;
  w &= keep;
  return keep != 0xffffffffu;
}
// 16 or 32 consecutive TMEM columns of this warp's 32 lanes; the registers may be used after
// tmem_landed() has named them.
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// (volatile statements keep their order: no use of the registers can move before the wait)
template <int W>
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[W]) {
#pragma unroll
  for (int n = 0; n < W; n++) asm volatile("" : "+r"(r[n]));
}
template <int W>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[W]) {
  tmem_get(taddr, r);
  tmem_wait_ld();
  tmem_landed(r);
}
__device__ __forceinline__ void tmem_store(uint32_t taddr, const uint32_t (&r)[32]) { tmem_st32(taddr, r); }
__device__ __forceinline__ void tmem_store(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st16(taddr, r); }

// The same as warp_wait, but the warp looks once, together, before it goes the long way (the softmax warps' meetings:
// eight trees 61.4 -> 60.8 us, fewer spills; the other waits did not gain).
__device__ __forceinline__ void warp_pass(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) (void)warp_wait(bar, parity, abort_flag, err);
}

// 1 in one lane of a converged warp (always the same one), 0 in the others.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
// D (+)= A B^T and the commit, by the lane for which `on` is not 0.  The instructions are predicated, not
// branched to, so that the warp's control flow stays uniform and the descriptors in uniform registers.
__device__ __forceinline__ void umma_if(uint32_t on, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// Reduces W (16 or 32) values per lane over the warp's lanes; value n's result in the lanes n % W.  Each
// step of the second loop hands half of the values to the lane at distance o and keeps the others.
template <int W, typename Op>
__device__ __forceinline__ float transpose_reduce(const float (&x)[W], Op op) {
  const int lane = threadIdx.x & 31;
  float v[W];
#pragma unroll
  for (int n = 0; n < W; n++) v[n] = x[n];
#pragma unroll
  for (int o = 16; o >= W; o >>= 1)
#pragma unroll
    for (int n = 0; n < W; n++) v[n] = op(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
#pragma unroll
  for (int o = W / 2; o >= 1; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int n = 0; n < o; n++) {
      const float give = up ? v[n] : v[n + o], keep = up ? v[n + o] : v[n];
      v[n] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  return v[0];
}

// Head dim d of `rows` query rows (from row gr0 of the kv head): adds the infinities and NaN of the V
// values that were taken out of the tile's stages from key0 on, for the rows that see their keys, to
// what this thread has just stored (in `part`, pitch floats from row to row, or in the output).
template <bool F32>
__device__ __noinline__ void add_non_finite(const TreeParams& p, Seq s, int b, int kvh, int key0, int k_end, int kfull,
                                            int d, int gr0, int rows, float* part, int pitch) {
  for (int key = key0; key < k_end; key++) {
    if (key >= kfull && key < s.base) {
      key = s.base - 1;
      continue;
    }
    const long long off = row_offset(p, b, kvh, key);
    if (off < 0) continue;
    const float v = __half2float(p.v[off + d]);
    if (fabsf(v) < INFINITY) continue;
    for (int n = 0; n < rows; n++) {
      const int gr = gr0 + n, t = gr / p.group;
      const Sees q = sees_of(p, s, t);
      if (!(key < s.base ? key >= q.kmin : ((q.bits >> (key - s.base)) & 1) != 0)) continue;
      const size_t at = ((size_t)(s.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group)) * p.hd + d;
      if (part != nullptr) {
        part[(size_t)n * pitch + d] += v;
      } else if constexpr (F32) {
        reinterpret_cast<float*>(p.out)[at] += v;
      } else {
        __half* o = reinterpret_cast<__half*>(p.out) + at;
        *o = __float2half_rn(__half2float(*o) + v);
      }
    }
  }
}

template <int HD, int N, bool F32, int R>
__global__ void __launch_bounds__(kThreadsTc, 1) tree_tc_kernel(const __grid_constant__ TreeParams p) {
  using C = Tc<HD, N, F32, R>;
  constexpr int MB = C::MB, ROWS = C::ROWS, W = C::W, UNITS = C::UNITS, NQ = C::NQ;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Sees* sees = reinterpret_cast<Sees*>(smem + C::OFF_SEES);
  float* scales = reinterpret_cast<float*>(smem + C::OFF_SCALE);
  uint32_t* okw = reinterpret_cast<uint32_t*>(smem + C::OFF_OK);
  // Only the loads walk through the list; the other roles read where a piece lies from here.
  Walk* pieces = reinterpret_cast<Walk*>(smem + C::OFF_INFO);
  static_assert(sizeof(Walk) <= 64, "piece ring");
  volatile int* badv = reinterpret_cast<volatile int*>(smem + C::OFF_BAD);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* landed = bars;              // [UNITS] 128 loading threads
  uint64_t* full = landed + UNITS;      // [UNITS] 3 handing-over warps
  uint64_t* empty = full + UNITS;       // [UNITS] MMA commit
  // A thread's plain arrival also says that what it stored before is there, which the arrivals of its copies do
  // not: pieces come with qlanded (and qfull), all that the softmax reads of a tile and a stage with sfull, badv
  // with pvdone.  (Barriers of their own for these cost the softmax a wait more in every stage: 32 chains 46.6
  // us, so 44.2.)
  uint64_t* qlanded = empty + UNITS;    // [4] tile & 3: 128 loading threads, and the 4 loading warps
  uint64_t* qfull = qlanded + 4;        // [4] 3 handing-over warps
  uint64_t* qempty = qfull + 4;         // [2] MMA commit
  uint64_t* sfull = qempty + 2;         // [8] stage & 7: MMA commit, and the 4 loading warps
  uint64_t* sfree = sfull + 8;          // [2] softmax warps
  uint64_t* pvdone = sfree + 2;         // [8] stage & 7: MMA commit, and the 3 handing-over warps
  uint64_t* pfull = pvdone + 8;         // softmax warps
  uint64_t* ofree = pfull + 1;          // softmax warps
  uint64_t* mend = ofree + 1;           // MMA commit
  uint64_t* meet_bar = mend + 1;        // [shares] its 4 softmax warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_END);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_END + 4);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // ---- barriers and TMEM, before the wait for the preceding kernel
  if (tid == 0) {
    for (int u = 0; u < UNITS; u++) {
      mbar_init(&landed[u], 128);
      mbar_init(&full[u], 3);
      mbar_init(&empty[u], 1);
    }
    for (int u = 0; u < 4; u++) {
      mbar_init(&qlanded[u], 128 + 4);
      mbar_init(&qfull[u], 3);
    }
    for (int u = 0; u < 2; u++) {
      mbar_init(&qempty[u], 1);
      mbar_init(&sfree[u], kSoftWarps);
    }
    for (int u = 0; u < 8; u++) {
      mbar_init(&sfull[u], 1 + 4);
      mbar_init(&pvdone[u], 1 + 3);
    }
    mbar_init(pfull, kSoftWarps);
    mbar_init(ofree, kSoftWarps);
    mbar_init(mend, 1);
    for (int u = 0; u < kShares; u++) mbar_init(&meet_bar[u], 4);
    *abort_flag = 0;
    for (int u = 0; u < 8; u++) badv[u] = 0;
    for (int u = 0; u < 4; u++) pieces[u] = Walk{};  // (what a role reads that had to give up a wait)
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {  // one CTA per SM (shared memory), so the allocation never waits
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait_primary();
  pdl_launch_dependents();

  // ---- this CTA's stages.  (One without work goes through the roles with none and frees its TMEM
  // like the others.)
  Plan plan;
  Walk at = {};
  const int cta = (int)blockIdx.x;
  // (the table lies where P will)
  int2* table = reinterpret_cast<int2*>(smem + C::OFF_P);
  static_assert(C::P_BYTES >= kTable * (int)sizeof(int2), "table of sequences");
  const int2 own = lane < p.batch ? table_entry(p, lane) : make_int2(0, 0);
  if (p.batch > 32 && p.batch <= kTable) {
    for (int b = tid; b < p.batch; b += kThreadsTc) table[b] = table_entry(p, b);
    __syncthreads();
  }
  const int n_stages = deal(p, own, table, cta, (int)gridDim.x, plan, at);
  // No warp writes P before every warp has read the table: the two softmax shares meet nowhere else before
  // the first stage's P.
  if (p.batch > 32 && p.batch <= kTable) __syncthreads();
  if (warp == kMmaWarp + 3) {
    // the tiles whose first pieces lie here and that others go on with: one that begins with this
    // CTA's stages, one at their end
    Walk w = at;
    int done = 0;                  // stages before tile w
    long long base = plan.origin;  // where it begins, in the list with the leads
    for (int piece = 0; piece < 2; piece++) {
      Cut c = {};
      const int here = min(w.s.stages - w.j, n_stages - done);
      if (n_stages > 0 && w.j == 0 && here < w.s.stages && (piece == 0 || done > 0)) {
        c.parts = plan.run > 0 ? w.chunks : (int)(plan.owner(base + plan.lead + w.s.stages - 1) - cta) + 1;
        c.stride = plan.run > 0 ? 2 * w.s.tiles : 2;
        c.rows = min(ROWS, w.s.T * p.group - w.tile * ROWS);
        c.row0 = w.s.row0;
        c.kvh = w.kvh;
        c.first = w.tile * ROWS;
      }
      if (plan.run > 0 && w.chunks == 1) c.parts = 0;
      if (lane == 0) p.cuts[2 * cta + piece] = c;
      if (plan.run > 0) {
        done = 0;
        w.j = 1;  // (no second piece)
        continue;
      }
      while (done + (w.j_end - w.j) < n_stages) {
        done += w.j_end - w.j;
        base += plan.lead + w.s.stages;
        w.next_tile(p);
      }
    }
  }
  __syncwarp();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sbase = smem_u32(smem);
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return wait_or_abort(bar, parity & 1u, abort_flag, p.err, code);
  };

  if (warp >= kLoadWarp && warp < kMmaWarp) {
    // ------------------------------------------------------------------------------ loads
    regs_down<C::REGS_LOAD>();
    const int pw = warp - kLoadWarp;
    int issued = 0;  // units
    // A lane copies the 16-byte pieces k = lane % 8 of rows 32 pw + 4 it + lane / 8, it = 0..7; what it
    // needs of a stage's rows is looked up once and kept for all units of K and, later, of V.
    struct Rows {
      uint32_t at[8];  // the row's piece, in 16-byte units from the pool's start
      uint32_t ok;     // bit it: the row is there
    };
    const int k8 = (lane & 7) * 8;
    const uint32_t lane_dst = (uint32_t)(pw * 4096 + (lane >> 3) * 128);
    const uint32_t sw0 = (uint32_t)(((lane & 7) ^ (lane >> 3)) << 4), sw1 = sw0 ^ 64u;  // it even, odd
    auto load_units = [&](const Rows& rows, const __half* pool) {
#pragma unroll 1
      for (int u = 0; u < MB; u++) {
        const int slot = issued % UNITS;
        if (issued >= UNITS) {
          (void)wait(&empty[slot], (uint32_t)(issued / UNITS - 1), G4A_DEVERR_WAIT_EMPTY);
          __syncwarp();
        }
        const uint32_t dst = sbase + C::OFF_RING + slot * kUnit + lane_dst;
        const bool in0 = u * 128 + k8 < p.hd, in1 = u * 128 + 64 + k8 < p.hd;
#pragma unroll
        for (int it = 0; it < 8; it++) {
          const uint32_t to = dst + it * 512 + (it & 1 ? sw1 : sw0);
          const bool ok = (rows.ok >> it) & 1u;
          const __half* from = pool + (size_t)rows.at[it] * 8;
          cp16(to, from + (in0 ? u * 128 : 0), ok && in0);
          cp16(to + 16384, from + (in1 ? u * 128 + 64 : 0), ok && in1);
        }
        cp_arrive(&landed[slot]);  // when this thread's copies have landed
        issued++;
      }
    };
    Walk w = at;
    Rows rows = {}, rows_before = {};
    int tile_no = -1;  // tiles this CTA has begun
    // The tile's queries into Q buffer tile_no % NQ (copies under way when it returns), and after the
    // tile's first keys are under way too, what its rows see.  Lane k looks up row pw + 4 k of the tile.
    long long mine = -1;  // that row of q, in heads
    auto load_queries = [&]() {
      const int kvh = w.kvh, tile = w.tile;
      const int qb = tile_no % NQ;
      if (tile_no >= NQ) {
        (void)wait(&qempty[qb], (uint32_t)(tile_no / NQ - 1), G4A_DEVERR_WAIT_EMPTY);
        __syncwarp();
      }
      const int live = min(ROWS, w.s.T * p.group - tile * ROWS);
      constexpr int RW = ROWS / 4;
      const int r_mine = pw + 4 * lane, gr = tile * ROWS + r_mine, t = gr / p.group;
      mine = -1;
      if (lane < RW && r_mine < live)
        mine = (long long)(w.s.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group);
      constexpr int PC = HD / 8;                  // 16-byte pieces of a row
      constexpr int PER = PC < 32 ? 32 / PC : 1;  // rows per copy instruction
      const uint32_t qa = sbase + qb * C::Q_BYTES;
#pragma unroll 4
      for (int k0 = 0; k0 < RW; k0 += PER) {
        const int kr = k0 + (PC < 32 ? lane / PC : 0), r = pw + 4 * kr;
        const long long o = __shfl_sync(0xffffffffu, mine, kr);
#pragma unroll
        for (int term = 0; term < (F32 ? 2 : 1); term++)
#pragma unroll
          for (int u = 0; u < (PC > 32 ? PC / 32 : 1); u++) {
            const int k = (PC < 32 ? lane % PC : lane + 32 * u), n = r + term * ROWS;
            // f32: the row's two f16 terms, [token, head][2][HD], from tree_split_kernel
            const bool ok = o >= 0 && (F32 || k * 8 < p.hd);
            const __half* src = F32 ? p.q_terms + ((size_t)(ok ? o : 0) * 2 + term) * HD
                                    : reinterpret_cast<const __half*>(p.q) + (size_t)(ok ? o : 0) * p.hd;
            cp16(qa + (k >> 3) * (N * 128) + n * 128 + (((k & 7) ^ (n & 7)) << 4), src + (ok ? k * 8 : 0), ok);
          }
      }
    };
    auto finish_queries = [&]() {
      constexpr int RW = ROWS / 4;
      const int sb = tile_no & 3, r_mine = pw + 4 * lane;
      if (pw == 0 && lane == 0) pieces[sb] = w;
      if (lane < RW) {
        Sees v = {0, ~0ull};  // rows past the last one: their results are not written
        if (mine >= 0) v = sees_of(p, w.s, (w.tile * ROWS + r_mine) / p.group);
        sees[sb * ROWS + r_mine] = v;
        if constexpr (F32) scales[sb * ROWS + r_mine] = mine >= 0 ? p.q_scale[mine] : 0.f;
      }
      cp_arrive(&qlanded[sb]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&qlanded[sb]);
    };
    for (int i = 0; i <= n_stages; i++) {
      if (i < n_stages) {
        const bool first = i == 0 || w.j == 0;
        if (first) tile_no++;
        if (first) load_queries();
        long long off = -1;
        const int key = w.key0() + pw * 32 + lane;
        if (key < w.s.L) off = row_offset(p, w.b, w.kvh, key);
        const uint32_t there = __ballot_sync(0xffffffffu, off >= 0);
        // (the ring holds at most five units, so the loads are less than eight stages ahead of the softmax, and no
        // phase of sfull or pvdone is passed while it is still waited for)
        if (lane == 0) okw[(i & 7) * 4 + pw] = there;
        rows.ok = 0;
#pragma unroll
        for (int it = 0; it < 8; it++) {
          const int r = it * 4 + (lane >> 3);
          const long long o = __shfl_sync(0xffffffffu, off, r);
          rows.at[it] = o >= 0 ? (uint32_t)((o + k8) >> 3) : 0u;
          rows.ok |= (o >= 0 ? 1u : 0u) << it;
        }
        load_units(rows, p.k);
        if (first) finish_queries();
        if (lane == 0) mbar_arrive(&sfull[i & 7]);
      }
      if (i > 0) load_units(rows_before, p.v);
      rows_before = rows;
      if (++w.j == w.j_end && i + 1 < n_stages) w.next_tile(p);
    }
    // No copy and no arrival of one may be under way when the CTA ends, also after an abort, when nobody
    // else waits for them (all four warps issue every unit, so these waits end).
    cp_wait_all();
    for (int u = 0; u < UNITS && u < issued; u++)
      (void)mbar_wait_bounded(&landed[u], (uint32_t)((issued - 1 - u) / UNITS) & 1u, p.err, G4A_DEVERR_WAIT_MMA);
    for (int u = 0; u < 4 && u <= tile_no; u++)
      (void)mbar_wait_bounded(&qlanded[u], (uint32_t)((tile_no - u) >> 2) & 1u, p.err, G4A_DEVERR_WAIT_MMA);
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------------------------ MMAs
    regs_down<C::REGS_MMA>();
    if (warp == kMmaWarp) {
      // The whole warp runs the loop and one elected lane's MMAs are predicated on: the control flow is
      // uniform, so descriptors stay in uniform registers.  With a loop that only lane 0 entered, or a
      // branch around the MMAs, the other warps' work slowed their issue to 110-130 cycles each; so
      // issued they run at 48 (N = 64), whatever the loads and the softmax do.
      const uint32_t on = elect_one();
      constexpr uint32_t idesc_s = f16_idesc(N, false), idesc_o = f16_idesc(N, true, true);
      auto ready = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity & 1u, abort_flag, p.err); };
      const uint64_t dp = sw128_desc(sbase + C::OFF_P, 16384, 1024);
      int slot = 0, tile_no = -1, tile_o = -1, j = 0, j_end = 0;
      uint32_t round = 0;  // of the ring
      bool first_prev = false, ok = true;
      for (int i = 0; ok && i <= n_stages; i++) {
        bool first = false;
        if (i < n_stages) {
          const int b = i & 1;
          first = j == j_end;
          if (first) {
            tile_no++;
            ok = ready(&qfull[tile_no & 3], (uint32_t)(tile_no >> 2));
            j = pieces[tile_no & 3].j;
            j_end = pieces[tile_no & 3].j_end;
          }
          const bool last = i + 1 == n_stages || ++j == j_end;
          if (ok && i >= 2) ok = ready(&sfree[b], (uint32_t)(i / 2 - 1));
          const uint64_t dq = sw128_desc(sbase + (tile_no % NQ) * C::Q_BYTES, 16, 1024);
          const uint32_t d = tmem + C::COL_S + (uint32_t)(b * N);
#pragma unroll 1
          for (int u = 0; u < MB; u++) {
            if (ok) ok = ready(&full[slot], round);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dk = sw128_desc(sbase + C::OFF_RING + slot * kUnit, 16, 1024);
            const uint64_t dqu = dq + (uint64_t)((u * 2 * N * 128) >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; kk++)
              umma_if(on, d, dk + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                            dqu + (uint64_t)(((kk >> 2) * (N * 128) + (kk & 3) * 32) >> 4), idesc_s,
                            kk > 0 ? 1u : u > 0 ? 1u : 0u);
            commit_if(on, &empty[slot]);
            if (u == MB - 1) {
              commit_if(on, &sfull[i & 7]);
              if (last) commit_if(on, &qempty[tile_no % NQ]);
            }
            if (++slot == UNITS) slot = 0, round++;
          }
          if (!ok) break;
        }
        if (i > 0) {  // O of stage i - 1
          if (first_prev) {
            tile_o++;
            if (tile_o > 0) ok = ready(ofree, (uint32_t)(tile_o - 1));
          }
          if (ok) ok = ready(pfull, (uint32_t)(i - 1));
          const uint32_t go_on = first_prev ? 0u : 1u;
#pragma unroll 1
          for (int u = 0; u < MB; u++) {
            if (ok) ok = ready(&full[slot], round);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dv = sw128_desc(sbase + C::OFF_RING + slot * kUnit, 16384, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; kk++)
              umma_if(on, tmem + C::COL_O + (uint32_t)(u * N), dv + (uint64_t)((kk * 2048) >> 4),
                            dp + (uint64_t)((kk * 2048) >> 4), idesc_o, kk > 0 ? 1u : go_on);
            commit_if(on, &empty[slot]);
            if (u == MB - 1) commit_if(on, &pvdone[(i - 1) & 7]);
            if (++slot == UNITS) slot = 0, round++;
          }
          if (!ok) break;
        }
        first_prev = first;
      }
      // no MMA may still be running when TMEM is freed, also after an abort
      commit_if(on, mend);
      (void)mbar_wait_bounded(mend, 0, p.err, G4A_DEVERR_WAIT_MMA);
    }
    if (warp > kMmaWarp) {
      // ---------------------------------------------------------------------------- handing over
      // Takes the units in the order of their loads: waits until one has landed, makes the copies
      // (generic proxy) visible to the tensor core (async proxy), passes it on.  (The same fence
      // in the MMA thread held every unit up by several hundred cycles.)
      // V of keys that not every row sees: p = 0 times an infinite or NaN V would reach the rows
      // that do not.  Such values become 0 here, and the epilogue adds them to the rows that do.
      const int hw = warp - kMmaWarp - 1;
      Walk w = {}, before = {};
      int unit = 0, tile_no = -1, tile_before = 0;
      auto pass = [&](uint64_t* from, uint64_t* to, uint32_t parity) {
        (void)warp_wait(from, parity & 1u, abort_flag, p.err);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(to);
      };
      for (int i = 0; i <= n_stages; i++) {
        if (i < n_stages) {
          for (int u = 0; u < MB; u++, unit++)
            pass(&landed[unit % UNITS], &full[unit % UNITS], (uint32_t)(unit / UNITS));
          if (w.j == w.j_end) {
            tile_no++;
            pass(&qlanded[tile_no & 3], &qfull[tile_no & 3], (uint32_t)(tile_no >> 2));
            w = pieces[tile_no & 3];
          }
        }
        if (i > 0) {
          const bool mixed = !before.clean(p);
          for (int u = 0; u < MB; u++, unit++) {
            if (mixed) {
              (void)warp_wait(&landed[unit % UNITS], (uint32_t)(unit / UNITS) & 1u, abort_flag, p.err);
              const int k0 = before.key0(), a1 = before.kfull(p) - k0, b0 = before.s.base - k0, b1 = before.s.L - k0;
              unsigned char* x0 = smem + C::OFF_RING + (unit % UNITS) * kUnit;
              bool bad = false;
              for (int e = hw * 32 + lane; e < kKeysT * 16; e += 96) {
                const int r = e >> 4;
                if (!(r < a1 || (r >= b0 && r < b1))) continue;
                uint4* x = reinterpret_cast<uint4*>(x0 + ((e >> 3) & 1) * 16384 + r * 128 + ((e & 7) << 4));
                uint4 v = *x;
                if (clear_non_finite(v.x) | clear_non_finite(v.y) | clear_non_finite(v.z) | clear_non_finite(v.w)) {
                  *x = v;
                  bad = true;
                }
              }
              if (bad) badv[(tile_before + 1) & 7] = (tile_before + 1) & 0xffff;
            }
            pass(&landed[unit % UNITS], &full[unit % UNITS], (uint32_t)(unit / UNITS));
          }
          if (lane == 0) mbar_arrive(&pvdone[(i - 1) & 7]);
        }
        before = w;
        tile_before = tile_no;
        w.j++;
      }
    }
  } else {
    // ------------------------------------------------------------------------------ softmax
    regs_up<C::REGS_SOFT>();
    const int quarter = warp & 3, share = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    float* su = reinterpret_cast<float*>(smem + C::OFF_U) + warp * W;
    float* sf = reinterpret_cast<float*>(smem + C::OFF_F) + warp * W;
    // Row maxima and row sums meet in places of their own, so that a tile's first maxima may be written while
    // a slower warp still reads the sums of the tile before (a first stage takes no vote).  Two writes of one
    // place have a meeting between them that follows the reads of the earlier one.
    float* smax = reinterpret_cast<float*>(smem + C::OFF_MAX) + share * 4 * W;
    float* ssum = reinterpret_cast<float*>(smem + C::OFF_SUM) + share * 4 * W;
    int* votes = reinterpret_cast<int*>(smem + C::OFF_VOTE) + share * 8;
    // The share's four warps meet (a bounded wait like every other); what they wrote before is visible
    // after.  `votes` alternates between two sets, so that nobody writes what another still reads.
    uint32_t met = 0;
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&meet_bar[share]);
      warp_pass(&meet_bar[share], met & 1u, abort_flag, p.err);
      met++;
    };
    auto any_of = [&](bool pred) {
      const bool mine = __any_sync(0xffffffffu, pred);
      int* v = votes + (met & 1) * 4;
      if (lane == 0) v[quarter] = mine ? 1 : 0;
      meet();
      const int4 all = *reinterpret_cast<const int4*>(v);
      return (all.x | all.y | all.z | all.w) != 0;
    };
    // the product of stage i has been added to O
    auto wait_pv = [&](int i) { (void)warp_wait(&pvdone[i & 7], (uint32_t)(i >> 3) & 1u, abort_flag, p.err); };
    const int key_in = quarter * 32 + lane;  // this thread's key of a stage
    const int n_of = lane % W;               // the row whose maximum and sum this lane keeps
    unsigned char* prow = smem + C::OFF_P + key_in * 128;
    Walk w = {};
    int tile_no = -1, j_first = 0;
    float m;     // running maximum of row n_of of the share
    float l[W];  // this thread's keys' part of the row sums
    auto reset = [&]() {
      m = -INFINITY;
#pragma unroll
      for (int n = 0; n < W; n++) l[n] = 0.f;
      __syncwarp();
      if (lane < W) su[lane] = kUnseen;
      __syncwarp();
    };
    reset();
    for (int i = 0; i < n_stages; i++) {
      const int b = i & 1;
      const bool first = w.j == w.j_end;
      (void)warp_wait(&sfull[i & 7], (uint32_t)(i >> 3) & 1u, abort_flag, p.err);
      tc_fence_after();
      if (first) {
        tile_no++;
        w = pieces[tile_no & 3];
        // (after an abort the loads run ahead and the piece may be half of another one: write nothing)
        if (*abort_flag) w.s.T = 0;
        j_first = w.j;
      }
      const bool last = i + 1 == n_stages || w.j + 1 == w.j_end;
      const int kvh = w.kvh, tile = w.tile;
      const int live = min(ROWS, w.s.T * p.group - tile * ROWS) - share * W;  // rows of this share
      if (live > 0) {
        const int key0 = w.key0(), key = key0 + key_in;
        const uint4 ok4 = *reinterpret_cast<const uint4*>(okw + (i & 7) * 4);
        const bool clean = w.clean(p) && (ok4.x & ok4.y & ok4.z & ok4.w) == ~0u;
        // ---- scores in powers of two
        float x[W];
        {
          uint32_t r[W];
          const uint32_t col = lanes + C::COL_S + (uint32_t)(b * N + share * W);
          if constexpr (F32) {
            const float* sc = scales + (tile_no & 3) * ROWS + share * W;
            uint32_t r2[W];
            tmem_get(col, r);
            tmem_get(col + ROWS, r2);
            tmem_wait_ld();
            tmem_landed(r);
            tmem_landed(r2);
#pragma unroll
            for (int n = 0; n < W; n += 4) {
              const float4 c4 = *reinterpret_cast<const float4*>(sc + n);
              const float cs[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
              for (int e = 0; e < 4; e++)
                x[n + e] = (__uint_as_float(r[n + e]) + __uint_as_float(r2[n + e])) * cs[e];
            }
          } else {
            tmem_load(col, r);
#pragma unroll
            for (int n = 0; n < W; n++) x[n] = __uint_as_float(r[n]) * p.scale_log2;
          }
        }
        if (!clean) {
          const uint32_t okq = quarter == 0 ? ok4.x : quarter == 1 ? ok4.y : quarter == 2 ? ok4.z : ok4.w;
          const bool there = (okq >> lane) & 1u;
          const Sees* see = sees + (tile_no & 3) * ROWS + share * W;
#pragma unroll
          for (int n = 0; n < W; n++) {
            const Sees v = see[n];
            const bool in = key < w.s.base ? key >= v.kmin : ((v.bits >> (key - w.s.base)) & 1) != 0;
            if (!there || !in) x[n] = -INFINITY;
          }
        }
        // every score of this buffer is in registers
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfree[b]);
        // ---- does a score pass its row's maximum by 2^8?
        float far = -INFINITY;
        const float4* u4 = reinterpret_cast<const float4*>(su);  // m - 7 of the rows
#pragma unroll
        for (int n = 0; n < W; n += 4) {
          const float4 u = u4[n / 4];
          far = fmaxf(far, fmaxf(fmaxf(x[n] - u.x, x[n + 1] - u.y), fmaxf(x[n + 2] - u.z, x[n + 3] - u.w)));
        }
        bool pv_waited = i == 0;
        if (first || any_of(far > kPUp + kRaise)) {
          const float mine = transpose_reduce<W>(x, [](float a, float c) { return fmaxf(a, c); });
          if (lane < W) smax[quarter * W + lane] = mine;
          meet();
          const float mx = fmaxf(fmaxf(smax[n_of], smax[W + n_of]), fmaxf(smax[2 * W + n_of], smax[3 * W + n_of]));
          const bool raise = mx > m + kRaise;
          const float f = !raise ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - mx);
          if (raise) m = mx;
          if (lane < W) {
            su[lane] = m == -INFINITY ? kUnseen : m - kPUp;
            sf[lane] = f;
          }
          __syncwarp();
#pragma unroll
          for (int n = 0; n < W; n++) l[n] *= sf[n];
          if (!first && __any_sync(0xffffffffu, f != 1.f)) {  // the same in the share's four warps
            wait_pv(i - 1);
            pv_waited = true;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < MB * (F32 ? 2 : 1); k++) {  // M blocks (x terms)
              const uint32_t col = lanes + C::COL_O + (uint32_t)((k % MB) * N + (k / MB) * ROWS + share * W);
              uint32_t r[W];
              tmem_load(col, r);
#pragma unroll
              for (int n = 0; n < W; n++) r[n] = __float_as_uint(__uint_as_float(r[n]) * sf[n]);
              tmem_store(col, r);
            }
            tmem_wait_st();
          }
        }
        // ---- p = 2^(s - m + 7)
        uint32_t hi[W / 2], lo[F32 ? W / 2 : 1];
#pragma unroll
        for (int n = 0; n < W; n += 4) {
          const float4 u = u4[n / 4];
          const float p0 = fast_exp2(x[n] - u.x), p1 = fast_exp2(x[n + 1] - u.y);
          const float p2 = fast_exp2(x[n + 2] - u.z), p3 = fast_exp2(x[n + 3] - u.w);
          l[n] += p0;
          l[n + 1] += p1;
          l[n + 2] += p2;
          l[n + 3] += p3;
          hi[n / 2] = pack2(p0, p1);
          hi[n / 2 + 1] = pack2(p2, p3);
          if constexpr (F32) {
            const float2 h0 = h2_to_f2(hi[n / 2]), h1 = h2_to_f2(hi[n / 2 + 1]);
            lo[n / 2] = pack2(p0 - h0.x, p1 - h0.y);
            lo[n / 2 + 1] = pack2(p2 - h1.x, p3 - h1.y);
          }
        }
        // the previous stage's product has read P
        if (!pv_waited) wait_pv(i - 1);
#pragma unroll
        for (int term = 0; term < (F32 ? 2 : 1); term++) {
          const int n0 = term * ROWS + share * W;  // first column of this thread's run
#pragma unroll
          for (int k = 0; k < W / 8; k++) {
            const int piece = n0 / 8 + k;
            const uint32_t* v = (term ? lo : hi) + 4 * k;
            *reinterpret_cast<uint4*>(prow + (piece >> 3) * 16384 + (((piece & 7) ^ (key_in & 7)) << 4)) =
                make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      } else {
        // no rows of the tile in this share: its columns' P is never looked at
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfree[b]);
        if (i > 0) wait_pv(i - 1);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull);

      if (last) {
        // ---- row sums, then O / l (or the part of a tile that other CTAs share)
        const bool whole = w.chunks == 1 && j_first == 0 && w.j + 1 == w.s.stages;
        const bool later = i - (w.j - j_first) > 0;  // not the piece this CTA's stages begin with
        float* part = p.part + ((size_t)2 * cta + (later ? 1 : 0)) * ROWS * (HD + 2);
        if (live > 0) {
          const float mine = transpose_reduce<W>(l, [](float a, float c) { return a + c; });
          if (lane < W) ssum[quarter * W + lane] = mine;
          meet();
          const float lt = (ssum[n_of] + ssum[W + n_of]) + (ssum[2 * W + n_of] + ssum[3 * W + n_of]);
          if (lane < W) sf[lane] = !whole ? 1.f : lt == 0.f ? 0.f : 1.f / lt;
          if (!whole && quarter == 0 && lane < W) {
            part[(size_t)ROWS * HD + share * W + lane] = m;
            part[(size_t)ROWS * HD + ROWS + share * W + lane] = lt;
          }
          __syncwarp();
        }
        wait_pv(i);
        tc_fence_after();
        if (live > 0) {
          const bool bad = badv[(tile_no + 1) & 7] == ((tile_no + 1) & 0xffff);
          const int nl = min(W, live);
          long long row = 0;  // lane n: where row n of the share lies in the output
          if (lane < nl) {
            const int gr = tile * ROWS + share * W + lane, t = gr / p.group;
            row = ((long long)(w.s.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group)) * p.hd;
          }
#pragma unroll 1
          for (int mb = 0; mb < MB; mb++) {
            const int d = mb * 128 + key_in;
            const uint32_t col = lanes + C::COL_O + (uint32_t)(mb * N + share * W);
            float o[W];
            {
              uint32_t r[W];
              if constexpr (F32) {
                uint32_t r2[W];
                tmem_get(col, r);
                tmem_get(col + ROWS, r2);
                tmem_wait_ld();
                tmem_landed(r);
                tmem_landed(r2);
#pragma unroll
                for (int n = 0; n < W; n++) o[n] = __uint_as_float(r[n]) + __uint_as_float(r2[n]);
              } else {
                tmem_load(col, r);
#pragma unroll
                for (int n = 0; n < W; n++) o[n] = __uint_as_float(r[n]);
              }
            }
            if (whole) {
#pragma unroll
              for (int n = 0; n < W; n++) {
                const long long a = __shfl_sync(0xffffffffu, row, n);
                if (n < nl && d < p.hd) {
                  const float y = o[n] * sf[n];
                  if constexpr (F32) reinterpret_cast<float*>(p.out)[a + d] = y;
                  else reinterpret_cast<__half*>(p.out)[a + d] = __float2half_rn(y);
                }
              }
            } else {
#pragma unroll
              for (int n = 0; n < W; n++)
                if (n < nl) part[(size_t)(share * W + n) * HD + d] = o[n];
            }
            if (bad && d < p.hd)
              add_non_finite<F32>(p, w.s, w.b, kvh, w.s.lo + j_first * kKeysT, min(w.key0() + kKeysT, w.s.L), w.kfull(p),
                                  d, tile * ROWS + share * W, nl, whole ? nullptr : part + (size_t)share * W * HD, HD);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ofree);
        reset();
      }
      w.j++;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
}

// f32 queries as two f16 terms and a scale, one warp per (token, head): x 2^e = hi + lo with the
// largest element brought to [2^10, 2^11), so that the low terms of every element that counts stay
// above f16's smallest step.  terms [token, head][2][hd_pad], zero beyond head_dim; scale = scale
// log2(e) 2^-e.  Once per call: inside the attention kernel every CTA of a long context would split
// the same rows again (10 us of its start at 64 rows).
__global__ void __launch_bounds__(256) tree_split_kernel(const float* q, __half* terms, float* scales, long long rows,
                                                         int hd, int hd_pad, float scale_log2) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_wait_primary();
  pdl_launch_dependents();
  if (row >= rows) return;
  float4 x[4];
  float big = 0.f;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int d = u * 128 + lane * 4;
    x[u] = d < hd ? *reinterpret_cast<const float4*>(q + row * hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    big = fmaxf(big, fmaxf(fmaxf(fabsf(x[u].x), fabsf(x[u].y)), fmaxf(fabsf(x[u].z), fabsf(x[u].w))));
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  int e = 0;
  if (big > 0.f && big < INFINITY) e = max(-120, min(120, 137 - (int)(__float_as_uint(big) >> 23)));
  const float up = __int_as_float((127 + e) << 23);
  if (lane == 0) scales[row] = ldexpf(scale_log2, -e);
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int d = u * 128 + lane * 4;
    if (d >= hd_pad) continue;
    const float v[4] = {x[u].x * up, x[u].y * up, x[u].z * up, x[u].w * up};
    float lo[4];
#pragma unroll
    for (int k = 0; k < 4; k++) lo[k] = v[k] - __half2float(__float2half_rn(v[k]));
    __half* to = terms + row * 2 * hd_pad + d;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    *reinterpret_cast<uint2*>(to + hd_pad) = make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
  }
}

template <int HD, int N, bool F32, int R>
g4a_status launch_tc(g4a_ctx* ctx, TreeParams& p, long long keys, long long tokens_rows) {
  using C = Tc<HD, N, F32, R>;
  static std::atomic<bool> done[64];
  if (ctx->device >= 64 || !done[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(tree_tc_kernel<HD, N, F32, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)C::SMEM);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(tree_tc_kernel)");
    if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
  }
  p.rows_log2 = C::ROWS == 64 ? 6 : 5;
  static_assert(C::ROWS == 64 || C::ROWS == 32, "tile rows");
  static_assert(C::ROWS * (F32 ? 2 : 1) <= N, "columns");
  p.hd_pad = HD;
  const long long tiles = (tokens_rows + C::ROWS - 1) / C::ROWS;
  const double stages = (double)(keys / kKeysT + p.batch) * (double)tiles * p.nkh;
  p.grid = (int)std::max(1.0, std::min(stages, (double)std::min(ctx->num_sms, kMaxGrid)));
  const size_t parts = (size_t)2 * p.grid * C::ROWS * (HD + 2) * sizeof(float);
  // workspace: the parts of cut tiles, the cuts, the queries' terms and scales (16-byte pieces)
  const size_t cuts = ((size_t)2 * p.grid * sizeof(Cut) + 15) & ~size_t(15);
  const size_t rows = F32 ? (size_t)p.tokens * p.nqh : 0, terms = rows * 2 * HD * sizeof(__half);
  const size_t need = parts + cuts + terms + rows * sizeof(float);
  if (g4a_status s = g4a_ensure_workspace(ctx, need)) return s;
  char* ws = static_cast<char*>(ctx->workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.cuts = reinterpret_cast<Cut*>(ws + parts);
  g4a_prof_scope ps(ctx, G4A_PROF_TREE_ATTN);
  if constexpr (F32) {
    __half* q_terms = reinterpret_cast<__half*>(ws + parts + cuts);
    float* q_scale = reinterpret_cast<float*>(ws + parts + cuts + terms);
    p.q_terms = q_terms;
    p.q_scale = q_scale;
    if ((rows + 7) / 8 > 0x7fffffffull) return g4a_fail(G4A_EINVAL, "g4a_tree_attn_paged: num_tokens * num_q_heads too large");
    const cudaError_t e = g4a_launch(tree_split_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, ctx->stream, true,
                                     static_cast<const float*>(p.q), q_terms, q_scale, (long long)rows, p.hd, HD,
                                     p.scale_log2);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch tree_split_kernel");
  }
  const cudaError_t e =
      g4a_launch(tree_tc_kernel<HD, N, F32, R>, dim3(p.grid), dim3(kThreadsTc), C::SMEM, ctx->stream, true, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch tree_tc_kernel");
  return G4A_OK;
}

}  // namespace

// Tile heights.  32 rows (64 columns; f16 queries leave half of them idle) where a sequence has no more or
// where that makes at most two stages for each SM: a softmax warp then has 16 rows instead of 32, and a
// CTA's softmax and epilogue are half as long.  64 rows beyond (f32 queries of up to 256 dims: 128 columns),
// which read and load each key for twice the rows.  Both sides measured, 32 / 64 rows: f32, 24 tokens x 8
// heads of 256 dims, 1,024 keys 16.9 / 20.1 us, 6,000 keys 20.7 / 28.7; 8 tokens over 32k keys (3.5 stages) 27
// / 27; 64 tokens over 32k 85 / 71.  f16, 7 tokens x 3 heads, 32 sequences 44 / 56; 24 tokens x 8 heads, 3,000
// keys 16.4 / 18.0.  (A head of more than 256 dims has room for 64 columns only, so f32 has 32 rows.)
g4a_status g4a_tree_tc_launch(g4a_ctx* ctx, g4a_tree::TreeParams& p, bool f32, long long keys) {
  const long long rows = (long long)p.max_tokens * p.group;
  const bool narrow =
      rows <= 32 || (double)(keys / kKeysT + p.batch) * (double)((rows + 31) / 32) * p.nkh <= 2.0 * ctx->num_sms;
  if (p.hd > 256) {
    if (f32) return launch_tc<512, 64, true, 32>(ctx, p, keys, rows);
    return narrow ? launch_tc<512, 64, false, 32>(ctx, p, keys, rows) : launch_tc<512, 64, false, 64>(ctx, p, keys, rows);
  }
  if (p.hd > 128) {
    if (f32)
      return narrow ? launch_tc<256, 64, true, 32>(ctx, p, keys, rows) : launch_tc<256, 128, true, 64>(ctx, p, keys, rows);
    return narrow ? launch_tc<256, 64, false, 32>(ctx, p, keys, rows) : launch_tc<256, 64, false, 64>(ctx, p, keys, rows);
  }
  if (f32)
    return narrow ? launch_tc<128, 64, true, 32>(ctx, p, keys, rows) : launch_tc<128, 128, true, 64>(ctx, p, keys, rows);
  return narrow ? launch_tc<128, 64, false, 32>(ctx, p, keys, rows) : launch_tc<128, 64, false, 64>(ctx, p, keys, rows);
}
