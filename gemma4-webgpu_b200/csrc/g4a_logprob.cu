// Log probabilities, entropy and top alternatives of logit rows (no reference counterpart: the
// reference samples on the host from the logits it reads back).
//
// Over one row, y = c tanh(x / c) (or x), m = max y, S = sum e^(y - m), T = sum (y - m) e^(y - m):
//   log p(t) = y_t - m - ln S,   H = ln S - T / S.
// All three fold over parts of the row: a part's S and T are rescaled to a larger m by
// S' = w S, T' = w (T + (m - m') S), w = e^(m - m').  So one pass over the logits is enough, split
// over as many CTAs as the batch leaves free; a second kernel joins the parts of a row.
//
// Top k.  Values are ranked by 64-bit keys (order-preserving bits of x above the complement of the
// id), so no two are equal and ties go to the lower id.  The pass over the logits only keeps the
// largest value of every segment of 512 consecutive ids (a warp's share of a tile; 1/512 of the
// row).  The join then takes the k + 2 largest segments, by (largest value, lower segment first),
// and looks for the k largest values in those alone: a value outside has k segments before its own
// whose largest values all rank above it.  (Two more than k because the first and the last segment
// of a row may be filled up with -inf.)
//
// Both selections are the same block-wide routine: tiles of 4,096 values against a sorted list of the
// best so far.  When more threads than wanted hold a value above the list's last, the k-th largest
// of the 256 thread maxima is a second lower bound (k values at least that large exist), so at most
// k threads append their 16 values and the list stays within k + 16 k for any input, equal values
// included.
#include <string.h>

#include "g4a_internal.cuh"

namespace {

constexpr int kThreadsL = 256;
constexpr int kMaxTop = G4A_MAX_TOP_K;
constexpr int kEpt = 16;                          // values per thread and tile
constexpr int kTile = kThreadsL * kEpt;
constexpr int kSeg = 32 * kEpt;                   // values of a segment
constexpr int kMaxPick = kMaxTop + 2;             // segments looked at
constexpr int kList = kMaxPick + kMaxPick * kEpt; // the kept values and those a tile appends
constexpr int kMaxSplit = kThreadsL;              // parts of a row: one thread each in the join
constexpr float kLog2eL = 1.4426950408889634f;
constexpr float kLn2L = 0.6931471805599453f;
// Caps up to this size bound a row's maximum so that m log2(e) is rounded by 2^-14 at most, and a first-order
// correction of the sums leaves less than 2^-29 of that.
constexpr float kNearCap = 1024.f;

struct LogprobParams {
  const void* logits;
  const int* tokens;
  size_t row_stride;
  uint32_t rows, vocab, split, part;  // part: values of a row per CTA (a multiple of kTile)
  int tokens_per_row, top_k;
  float cap, inv_cap, inv_cap2;  // inv_cap2 = 2 log2(e) / cap
  float4* stats;                 // [rows, split] (m, S, T)
  float* seg_max;                // [rows, segs]
  uint32_t segs;
  float *logprob, *entropy, *top_logprob;
  int* top_ids;
  int* err;
};

// Order-preserving bits: larger floats give larger words, -0 = +0, NaN below everything.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  if (o == 0u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t make_key(float x, uint32_t id) {
  return ((uint64_t)ordered(x) << 32) | (0xffffffffu - id);
}

// c tanh(x / c) = c (1 - 2 / (e^(2x/c) + 1)); the exponential's overflow and underflow give +-c.
// The absolute error is a few ulp of c, a few 1e-6 at c = 30: the size of a logit's own rounding.
// -inf (a banned token, and the filler of values outside the row) stays -inf.
__device__ __forceinline__ float capped(float x, float cap, float inv_cap2) {
  const float e = g4a::fast_exp2(x * inv_cap2);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
  const float y = fmaf(-2.0f * cap, r, cap);
  return x == -INFINITY ? -INFINITY : y;
}

// The same for |x| <= 0.9 c as x times a polynomial in (x / c)^2, a least-maximum fit of tanh(z) / z on
// [0, 0.9] (relative error 1.4e-8): nine multiply-adds where the form above takes two special-
// function operations, of which an SM makes 16 a cycle against 128 of the former.
constexpr float kCapRange = 0.9f;
constexpr float kT0 = 0.99999998584f, kT1 = -0.33333160193f, kT2 = 0.13329835261f, kT3 = -0.05369905191f,
                kT4 = 0.02085770253f, kT5 = -0.00681405711f, kT6 = 0.00128645157f;
__device__ __forceinline__ float capped_small(float x, float inv_cap) {
  const float z = x * inv_cap, u = z * z;
  float q = kT6;
  q = fmaf(q, u, kT5);
  q = fmaf(q, u, kT4);
  q = fmaf(q, u, kT3);
  q = fmaf(q, u, kT2);
  q = fmaf(q, u, kT1);
  q = fmaf(q, u, kT0);
  return x * q;
}

// Which of the two, by the value alone: the parts and the join have to agree, so that what a logit's own
// rounding adds to log p cancels where it is the largest.
__device__ __forceinline__ float capped_by(float x, float cap, float inv_cap, float inv_cap2) {
  return fabsf(x) <= kCapRange * cap ? capped_small(x, inv_cap) : capped(x, cap, inv_cap2);
}

// Two floats in one 64-bit register: the packed multiply-add does both in one issue slot (384 capped rows of
// 262,144: 101 us with single ones, 87 so).
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// capped_small of two values
__device__ __forceinline__ uint64_t capped_small2(uint64_t x, uint64_t inv_cap) {
  const uint64_t z = mul2(x, inv_cap), u = mul2(z, z);
  uint64_t q = two(kT6, kT6);
  q = fma2(q, u, two(kT5, kT5));
  q = fma2(q, u, two(kT4, kT4));
  q = fma2(q, u, two(kT3, kT3));
  q = fma2(q, u, two(kT2, kT2));
  q = fma2(q, u, two(kT1, kT1));
  q = fma2(q, u, two(kT0, kT0));
  return mul2(x, q);
}

// Largest of a warp's values, in one instruction (NaN is passed over).
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

struct Stat {
  float m, s, t;  // t in log2 units: sum (y - m) log2(e) e^(y - m)
};
__device__ __forceinline__ Stat join(const Stat a, const Stat b) {
  const float m = fmaxf(a.m, b.m);
  Stat r = {m, 0.f, 0.f};
  // a part with nothing in it (m = -inf) has s = t = 0 unless it met a NaN, which has to stay
  const float da = a.m == -INFINITY ? 0.f : (a.m - m) * kLog2eL, db = b.m == -INFINITY ? 0.f : (b.m - m) * kLog2eL;
  const float wa = g4a::fast_exp2(da), wb = g4a::fast_exp2(db);
  r.s = wa * a.s + wb * b.s;
  r.t = (wa > 0.f ? wa * (a.t + da * a.s) : 0.f) + (wb > 0.f ? wb * (b.t + db * b.s) : 0.f);
  return r;
}
__device__ __forceinline__ Stat block_join(Stat x, Stat* red) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const Stat y = {__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.s, o),
                    __shfl_xor_sync(0xffffffffu, x.t, o)};
    x = join(x, y);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = red[threadIdx.x & (kThreadsL / 32 - 1)];
#pragma unroll
  for (int o = kThreadsL / 64; o >= 1; o >>= 1) {
    const Stat y = {__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.s, o),
                    __shfl_xor_sync(0xffffffffu, x.t, o)};
    x = join(x, y);
  }
  return x;
}

// The k largest of n keys into kept[0, k), sorted, 0 where there are fewer; key(i) gives the i-th (0:
// none).  All 256 threads; `low`: values below this key are known not to be among them.  A barrier first:
// where the count of a list that did not fit led here, every thread has read it before it is reset.
struct alignas(16) TopShared {
  uint64_t list[kList], kept[kMaxPick], tops[kThreadsL];
  uint64_t bound;
  int count;
};
template <typename Key>
__device__ __forceinline__ void block_top(uint64_t n, int k, uint64_t low, TopShared& sh, Key key) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < kMaxPick) sh.kept[tid] = 0;
  if (tid == 0) sh.count = 0;
  int have = 0;
  uint64_t lim0 = low > 1 ? low : 1;
  __syncthreads();
  for (uint64_t t0 = 0; t0 < n; t0 += kTile) {
    uint64_t x[kEpt], best = 0;
#pragma unroll
    for (int e = 0; e < kEpt; e++) {
      const uint64_t i = t0 + (uint32_t)(e * kThreadsL + tid);
      x[e] = i < n ? key(i) : 0;
    }
#pragma unroll
    for (int e = 0; e < kEpt; e++) best = x[e] > best ? x[e] : best;
    const bool holds = best >= lim0;
    const int n_hold = __syncthreads_count(holds);
    if (n_hold == 0) continue;
    uint64_t lim = lim0;
    if (n_hold > k) {
      sh.tops[tid] = holds ? best : 0;
      __syncthreads();
      if (holds) {
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < kThreadsL; j += 2) {
          const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.tops[j]);
          rank += (o.x > best) + (o.y > best);
        }
        if (rank == k - 1) sh.bound = best;
      }
      __syncthreads();
      lim = max(lim, sh.bound);
    }
    if (best >= lim) {
#pragma unroll
      for (int e = 0; e < kEpt; e++)
        if (x[e] >= lim) sh.list[atomicAdd(&sh.count, 1)] = x[e];
    }
    const uint64_t old = tid < have ? sh.kept[tid] : 0;
    __syncthreads();
    const int added = sh.count, all = added + have;
    if (tid < have) sh.list[added + tid] = old;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    for (int i = tid; i < all; i += kThreadsL) {
      const uint64_t mine = sh.list[i];
      int rank = 0;
      for (int j = 0; j < all; j++) rank += sh.list[j] > mine;
      if (rank < k) sh.kept[rank] = mine;
    }
    __syncthreads();
    have = min(all, k);
    if (have == k) lim0 = max(lim0, sh.kept[k - 1] + 1);
  }
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = g4a::h2_to_f2(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
};

// One part of one row: CTA (row, part).  A tile is 8 warps x 512 consecutive values (16 a thread), in
// 16-byte loads from the aligned address at or before the row's start; a segment that reaches over
// either end of the row is read value by value, so nothing outside the row is read.  No thread
// waits for another before the end of the part.
// 384 rows of 262,144 f32 logits, capped, with 8 alternatives: the call takes 78 us, 5.2 TB/s (0.79 of the
// measured copy), without the cap 68, without cap and alternatives 65 (0.95); f16 logits 75 and 48.  (In short runs;
// after 10 ms of them the power limit lowers the clock to 1,715 MHz and 78 becomes 89.)  Rows with banned tokens
// leave the packed sums where there is a cap: 120.  More CTAs to an SM (fewer
// registers), or more and shorter parts, were slower.  A few rows are bound by latency, the part's loads and
// the join's chain (one row 8.7 us, 37 odd f16 rows of 50,257 8.5).
// CAP: 0 no cap, 1 a cap of at most kNearCap, 2 a larger one.  With 1 the exponents are y log2(e) - ml, one
// multiply-add each, and what rounding left of m log2(e) in ml, the same for all values, is taken out of the
// sums: 2^-left s, 2^-left (t - left s).  Otherwise the maximum may be huge (a row of which a thread has seen
// tokens banned by a large negative value alone, say) and that remainder no small correction: the
// difference y - m comes first, so that the maximum's own exponent is 0.
template <typename T, int CAP>
__global__ void __launch_bounds__(kThreadsL) logprob_part_kernel(const LogprobParams p) {
  constexpr int VN = Vec<T>::N, NV = kEpt / VN;
  __shared__ Stat red[kThreadsL / 32];
  const uint32_t row = blockIdx.x / p.split, part = blockIdx.x - row * p.split;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();
  const T* x0 = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride;
  // ids are counted from the aligned address; ids below `head` lie before the row
  const uint32_t head = (uint32_t)((reinterpret_cast<uintptr_t>(x0) & 15u) / sizeof(T));
  const T* base = x0 - head;
  const uint32_t lo = max(part * p.part, head);
  const uint32_t hi = min(part * p.part + p.part, p.vocab + head);
  float* seg_max = p.top_k ? p.seg_max + (size_t)row * p.segs : nullptr;
  // values that the packed sums take: within the polynomial's range, or (no cap) with finite exponents
  const float small = CAP ? kCapRange * p.cap : 1.0e38f;
  Stat st = {-INFINITY, 0.f, 0.f};
  // the next segment's values are on their way while this one's are summed
  uint4 raw[NV];
  auto fetch = [&](uint32_t t0) {
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const uint32_t i0 = t0 + (uint32_t)(j * 32 + lane) * VN;
      if (i0 >= lo && i0 + VN <= hi) {
        raw[j] = __ldcs(reinterpret_cast<const uint4*>(base + i0));
      } else {  // over an end of the row: value by value, -inf outside
        T v[VN];
#pragma unroll
        for (int e = 0; e < VN; e++) v[e] = i0 + e >= lo && i0 + e < hi ? base[i0 + e] : (T)(-INFINITY);
        memcpy(&raw[j], v, 16);
      }
    }
  };
  const uint32_t first = part * p.part + warp * kSeg;
  if (first < hi) fetch(first);
  for (uint32_t t0 = first; t0 < hi; t0 += kTile) {
    float x[kEpt];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      float v[VN];
      Vec<T>::unpack(raw[j], v);
#pragma unroll
      for (int e = 0; e < VN; e++) x[j * VN + e] = v[e];
    }
    if (t0 + kTile < hi) fetch(t0 + kTile);
    float top = x[0], low = x[0];
#pragma unroll
    for (int e = 1; e < kEpt; e++) top = fmaxf(top, x[e]), low = fminf(low, x[e]);  // NaN is passed over
    if (seg_max != nullptr) {
      const float s = warp_max(top);
      if (lane == 0) seg_max[t0 / kSeg] = s;
    }
    const float ym = CAP ? capped_by(top, p.cap, p.inv_cap, p.inv_cap2) : top;
    const float m = fmaxf(st.m, ym);
    if (m > st.m) {
      const float d = st.m == -INFINITY ? 0.f : (st.m - m) * kLog2eL, w = g4a::fast_exp2(d);
      st.t = CAP == 1 || w > 0.f ? w * (st.t + d * st.s) : 0.f;  // (without a near cap d may be -inf)
      st.s *= w;
      st.m = m;
    }
    const float mf = m == -INFINITY ? 0.f : m, ml = mf * kLog2eL, left = fmaf(mf, kLog2eL, -ml);
    float s = 0.f, t = 0.f;
    if ((CAP ? top : m) <= small && low >= -small) {
      uint64_t s2 = 0, t2 = 0;
      const uint64_t ic = two(p.inv_cap, p.inv_cap), l2 = two(kLog2eL, kLog2eL);
      const uint64_t off = CAP == 1 ? two(-ml, -ml) : two(-m, -m);
#pragma unroll
      for (int e = 0; e < kEpt; e += 2) {
        const uint64_t x2 = two(x[e], x[e + 1]), y2 = CAP ? capped_small2(x2, ic) : x2;
        const uint64_t d2 = CAP == 1 ? fma2(y2, l2, off) : mul2(add2(y2, off), l2);
        float d0, d1;
        apart(d2, d0, d1);
        const uint64_t w2 = two(g4a::fast_exp2(d0), g4a::fast_exp2(d1));
        s2 = add2(s2, w2);
        t2 = fma2(d2, w2, t2);
      }
      float a, b;
      apart(s2, a, b);
      s = a + b;
      apart(t2, a, b);
      t = a + b;
    } else {
#pragma unroll
      for (int e = 0; e < kEpt; e++) {
        const float y = CAP ? capped_by(x[e], p.cap, p.inv_cap, p.inv_cap2) : x[e];
        const float d = CAP == 1 ? fmaf(y, kLog2eL, -ml) : (y - mf) * kLog2eL;
        const float w = g4a::fast_exp2(d);
        s += w;
        t = fmaf(fmaxf(d, -1000.f), w, t);  // -inf: -1000 * 0
      }
    }
    if constexpr (CAP == 1) {
      const float f = fmaf(-kLn2L, left, 1.0f);
      st.s = fmaf(f, s, st.s);
      st.t = fmaf(f, fmaf(-left, s, t), st.t);
    } else {
      st.s += s;
      st.t += t;
    }
  }
  st = block_join(st, red);
  if (tid == 0) p.stats[(size_t)row * p.split + part] = make_float4(st.m, st.s, st.t, 0.f);
}

// Joins the parts of one row (at most one per thread) and picks its largest values.
template <typename T>
__global__ void __launch_bounds__(kThreadsL) logprob_join_kernel(const LogprobParams p) {
  __shared__ Stat red[kThreadsL / 32];
  __shared__ TopShared sh;
  __shared__ uint32_t picked[kMaxPick];
  const uint32_t row = blockIdx.x;
  const int tid = threadIdx.x, k = p.top_k, ns = (int)p.split;
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();
  const T* x0 = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride;
  const uint32_t head = (uint32_t)((reinterpret_cast<uintptr_t>(x0) & 15u) / sizeof(T));
  const uint32_t segs = k ? (p.vocab + head + kSeg - 1) / kSeg : 0;
  const float* seg_max = p.seg_max + (size_t)row * p.segs;
  // every load that needs nothing else first
  constexpr int kNear = 4;  // segments per thread of a row of up to 1024
  float near[kNear];
#pragma unroll
  for (int e = 0; e < kNear; e++) near[e] = (uint32_t)(e * kThreadsL + tid) < segs ? seg_max[e * kThreadsL + tid] : 0.f;
  const int my_tok = tid < p.tokens_per_row ? p.tokens[(size_t)row * p.tokens_per_row + tid] : -1;
  Stat st = {-INFINITY, 0.f, 0.f};
  if (tid < ns) {
    const float4 f = p.stats[(size_t)row * ns + tid];
    st = {f.x, f.y, f.z};
  }
  const float my_x = my_tok >= 0 && (uint32_t)my_tok < p.vocab ? Vec<T>::one(x0 + my_tok) : 0.f;
  st = block_join(st, red);  // (a barrier inside)
  const float ln_s = logf(st.s);
  const float cap = p.cap;
  auto value = [&](float x) {  // log probability of a logit
    const float y = cap > 0.f ? capped_by(x, cap, p.inv_cap, p.inv_cap2) : x;
    return y - st.m - ln_s;
  };
  if (p.entropy && tid == 0) p.entropy[row] = ln_s - kLn2L * st.t / st.s;
  for (int j = tid; j < p.tokens_per_row; j += kThreadsL) {
    const int tok = j == tid ? my_tok : p.tokens[(size_t)row * p.tokens_per_row + j];
    float lp = 0.f;
    if (tok >= 0 && (uint32_t)tok < p.vocab) {
      lp = value(j == tid ? my_x : Vec<T>::one(x0 + tok));
    } else if (tok != -1) {
      lp = __uint_as_float(0x7fc00000u);
      atomicExch(p.err, G4A_DEVERR_TOKEN);
    }
    p.logprob[(size_t)row * p.tokens_per_row + j] = lp;
  }
  if (k == 0) return;
  const int pick = (int)min(segs, (uint32_t)k + 2);
  auto rank_list = [&](int all, int want) {  // the list's `want` largest into kept
    for (int i = tid; i < all; i += kThreadsL) {
      const uint64_t mine = sh.list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < all; j++) rank += sh.list[j] > mine;
      if (rank < want) sh.kept[rank] = mine;
    }
    __syncthreads();
  };
  // ---- the segments.  A row of up to 1024 of them: the pick-th largest of 64 maxima (of four threads'
  // segments each) bounds the pick-th segment from below; what reaches it, mostly not twice as many as
  // are wanted, is listed and ranked.  (Of all 256 thread maxima: a sharper bound, but 2.4 us of counting; a
  // call of one row took 10.4 us, takes 8.7.)
  bool have_segs = false;
  if (segs <= kNear * kThreadsL) {
    uint32_t o[kNear], best = 0;
#pragma unroll
    for (int e = 0; e < kNear; e++) {
      o[e] = (uint32_t)(e * kThreadsL + tid) < segs ? ordered(near[e]) : 0u;
      best = max(best, o[e]);
    }
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 1));
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 2));
    uint32_t* tops = reinterpret_cast<uint32_t*>(sh.tops);
    if ((tid & 3) == 0) tops[tid >> 2] = best;
    if (tid == 0) sh.bound = 0, sh.count = 0;
    __syncthreads();
    if (tid < kThreadsL / 4) {
      const uint32_t mine = tops[tid];
      int above = 0, equal = 0;
#pragma unroll
      for (int j = 0; j < kThreadsL / 16; j++) {
        const uint4 v = reinterpret_cast<const uint4*>(tops)[j];
        above += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
        equal += (v.x == mine) + (v.y == mine) + (v.z == mine) + (v.w == mine);
      }
      if (above < pick && pick <= above + equal) sh.bound = mine;
    }
    __syncthreads();
    const uint32_t bound = (uint32_t)sh.bound;
#pragma unroll
    for (int e = 0; e < kNear; e++)
      if ((uint32_t)(e * kThreadsL + tid) < segs && o[e] >= bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) sh.list[at] = ((uint64_t)o[e] << 32) | (0xffffffffu - (uint32_t)(e * kThreadsL + tid));
      }
    __syncthreads();
    const int all = sh.count;
    have_segs = all <= kList;
    if (have_segs) rank_list(all, pick);
  }
  if (!have_segs) block_top(segs, pick, 0, sh, [&](uint64_t i) { return make_key(seg_max[i], (uint32_t)i); });
  if (tid < pick) picked[tid] = 0xffffffffu - (uint32_t)sh.kept[tid];
  // the k-th segment's largest value bounds the k-th value from below (its id is not known here)
  const uint64_t low = pick == k + 2 ? (sh.kept[k + 1] >> 32) << 32 : 0;
  __syncthreads();
  const uint32_t n = (uint32_t)pick * kSeg;
  auto id_of = [&](uint32_t i) { return (long long)picked[i / kSeg] * kSeg + (long long)(i % kSeg) - head; };
  // Few values of the picked segments reach the bound (k and a handful): all of them are loaded at
  // once, those that do are listed and ranked.  If they do not fit (equal values), or there is no
  // bound (a short row), the general selection does it.
  bool listed = false;
  if (low != 0) {
    const float bound = from_ordered((uint32_t)(low >> 32));
    if (tid == 0) sh.count = 0;
    __syncthreads();
    constexpr int VN = Vec<T>::N, kFly = 6;  // 16-byte loads of a thread in flight
    constexpr uint32_t per_seg = kSeg / VN;
    const T* base = x0 - head;
    for (uint32_t v0 = tid; v0 < (uint32_t)pick * per_seg; v0 += kFly * kThreadsL) {
      uint4 raw[kFly];
      uint32_t first[kFly];  // its first id, from the aligned address
#pragma unroll
      for (int f = 0; f < kFly; f++) {
        const uint32_t v = v0 + f * kThreadsL;
        first[f] = 0xffffffffu;
        if (v >= (uint32_t)pick * per_seg) continue;
        first[f] = picked[v / per_seg] * kSeg + v % per_seg * VN;
        if (first[f] >= head && first[f] + VN <= p.vocab + head) {
          raw[f] = *reinterpret_cast<const uint4*>(base + first[f]);
        } else {
          T x[VN];
#pragma unroll
          for (int e = 0; e < VN; e++)
            x[e] = first[f] + e >= head && first[f] + e < p.vocab + head ? base[first[f] + e] : (T)(-INFINITY);
          memcpy(&raw[f], x, 16);
        }
      }
#pragma unroll
      for (int f = 0; f < kFly; f++) {
        if (first[f] == 0xffffffffu) continue;
        float x[VN];
        Vec<T>::unpack(raw[f], x);
#pragma unroll
        for (int e = 0; e < VN; e++)
          if (x[e] >= bound && first[f] + e >= head && first[f] + e < p.vocab + head) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.list[at] = make_key(x[e], first[f] + e - head);
          }
      }
    }
    __syncthreads();
    const int all = sh.count;
    listed = all <= kList;
    if (listed) rank_list(all, k);
  }
  if (!listed)
    block_top(n, k, low, sh, [&](uint64_t i) -> uint64_t {
      const long long id = id_of((uint32_t)i);
      return id >= 0 && id < (long long)p.vocab ? make_key(Vec<T>::one(x0 + id), (uint32_t)id) : 0;
    });
  if (tid < k) {
    const uint64_t key = sh.kept[tid];
    p.top_ids[(size_t)row * k + tid] = (int)(0xffffffffu - (uint32_t)key);
    p.top_logprob[(size_t)row * k + tid] = value(from_ordered((uint32_t)(key >> 32)));
  }
}

template <typename T>
g4a_status launch_logprobs(g4a_ctx* ctx, LogprobParams& p) {
  // parts of a row: enough CTAs to fill the SMs several times over, whole tiles each
  const uint32_t tiles = (p.vocab + 8 + kTile - 1) / kTile;  // + the values before an unaligned row
  const uint32_t want = (uint32_t)(ctx->num_sms * 16);
  uint32_t split = (want + p.rows - 1) / p.rows;
  split = split < 1 ? 1 : split > tiles ? tiles : split;
  if (split > (uint32_t)kMaxSplit) split = kMaxSplit;
  const uint32_t per = (tiles + split - 1) / split;
  p.split = (tiles + per - 1) / per;
  p.part = per * kTile;
  if ((uint64_t)p.rows * p.split > 0x7fffffffull)
    return g4a_fail(G4A_EINVAL, "g4a_token_logprobs: rows %u too many", p.rows);
  const size_t parts = (size_t)p.rows * p.split;
  p.segs = tiles * (kTile / kSeg);
  const size_t segs = p.top_k ? (size_t)p.rows * p.segs : 0;
  if (g4a_status s = g4a_ensure_workspace(ctx, parts * sizeof(float4) + segs * sizeof(float))) return s;
  p.stats = static_cast<float4*>(ctx->workspace);
  p.seg_max = reinterpret_cast<float*>(p.stats + parts);
  g4a_prof_scope ps(ctx, G4A_PROF_TOKEN_LOGPROBS);
  cudaError_t e = g4a_launch(p.cap > kNearCap ? logprob_part_kernel<T, 2>
                             : p.cap > 0.f    ? logprob_part_kernel<T, 1>
                                              : logprob_part_kernel<T, 0>,
                             dim3((unsigned)parts), dim3(kThreadsL), 0, ctx->stream, true, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch logprob_part_kernel");
  e = g4a_launch(logprob_join_kernel<T>, dim3(p.rows), dim3(kThreadsL), 0, ctx->stream, true, p);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch logprob_join_kernel");
  return G4A_OK;
}

}  // namespace

extern "C" g4a_status g4a_token_logprobs(g4a_ctx* ctx, const void* logits, uint32_t format, const int32_t* tokens,
                                         uint32_t rows, uint32_t vocab, uint64_t row_stride, uint32_t tokens_per_row,
                                         uint32_t top_k, float softcap, float* logprob, float* entropy,
                                         float* top_logprob, int32_t* top_ids) {
  G4A_CHECK_CTX(ctx);
  const char* fn = "g4a_token_logprobs";
  if (format != G4A_ACT_F32 && format != G4A_ACT_F16) return g4a_fail(G4A_EINVAL, "%s: unknown format %u", fn, format);
  if (rows == 0) return G4A_OK;
  if (!logits) return g4a_fail(G4A_EINVAL, "%s: null logits", fn);
  if (rows > 0x7fffffffu) return g4a_fail(G4A_EINVAL, "%s: rows %u too many", fn, rows);
  if (vocab == 0 || vocab > 0x7ffff000u) return g4a_fail(G4A_EINVAL, "%s: vocab %u out of range", fn, vocab);
  if (row_stride == 0) row_stride = vocab;
  if (row_stride < vocab) return g4a_fail(G4A_EINVAL, "%s: row_stride below vocab %u", fn, vocab);
  if ((uintptr_t)logits & (format == G4A_ACT_F32 ? 3u : 1u)) return g4a_fail(G4A_EINVAL, "%s: unaligned logits", fn);
  if (top_k > (uint32_t)kMaxTop || top_k > vocab)
    return g4a_fail(G4A_EINVAL, "%s: top_k %u exceeds %d or vocab %u", fn, top_k, kMaxTop, vocab);
  if (tokens_per_row > 0x7fffffffu) return g4a_fail(G4A_EINVAL, "%s: tokens_per_row out of range", fn);
  if (tokens_per_row && (!tokens || !logprob)) return g4a_fail(G4A_EINVAL, "%s: null tokens or logprob", fn);
  if (top_k && (!top_logprob || !top_ids)) return g4a_fail(G4A_EINVAL, "%s: null top_logprob or top_ids", fn);
  if (softcap != 0.f && !(softcap >= 1e-30f && softcap <= 1e30f))  // (its reciprocal has to be finite)
    return g4a_fail(G4A_EINVAL, "%s: softcap must be 0 or in [1e-30, 1e30]", fn);
  if (tokens_per_row == 0 && !entropy && top_k == 0) return G4A_OK;
  g4a_device_guard dev(ctx);
  if (dev.status != G4A_OK) return dev.status;
  LogprobParams p = {};
  p.logits = logits;
  p.tokens = tokens;
  p.row_stride = row_stride;
  p.rows = rows;
  p.vocab = vocab;
  p.tokens_per_row = (int)tokens_per_row;
  p.top_k = (int)top_k;
  p.cap = softcap;
  p.inv_cap = softcap > 0.f ? 1.0f / softcap : 0.f;
  p.inv_cap2 = softcap > 0.f ? 2.0f * kLog2eL / softcap : 0.f;
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_logprob = top_logprob;
  p.top_ids = top_ids;
  p.err = ctx->dev_err_dev;
  return format == G4A_ACT_F16 ? launch_logprobs<__half>(ctx, p) : launch_logprobs<float>(ctx, p);
}
