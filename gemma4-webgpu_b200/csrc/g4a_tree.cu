// Attention of drafted tokens over a paged cache (g4a_tree_attn_paged): every token of a tree sees
// the prefix and its own ancestors.  No reference counterpart; the semantics of one token are
// those of shaders/attn_score.wgsl, softmax.wgsl and attn_output.wgsl over the rows it sees.
//
// The T tokens x G q heads that share a kv head are T * G query rows over the same keys, so a
// tile of rows reads a key once for all of them.  One pass over the keys with a running row
// maximum m and sum l: p = 2^(s - m + 15), o = sum p v, l = sum p, both rescaled by 2^(m_old -
// m_new) when m grows; out = o / l.  Long key ranges are cut over the CTAs; the parts (m, l, o) of
// a tile that several CTAs computed are joined by tree_merge_kernel.
//
// Numbers.  The products run on the tensor cores with f16 operands and f32 sums.  K and V are f16.
// With f32 queries, q and p are each split into two f16 terms (x = hi + lo, lo = f16(x - hi)), 22
// bits together, which is f32's accuracy in all but the last two bits; a query row is scaled by a
// power of two first (its largest element to [2^10, 2^11)) and p carries the factor 2^15, so the
// low terms stay above f16's smallest step (2^-24) for every element that counts.  With f16 queries
// p is rounded once to f16 (the output is f16 too); the sum l is taken over the unrounded p.
#include <algorithm>
#include <atomic>

#include "g4a_tree.cuh"

namespace {

using namespace g4a_tree;

constexpr int kThreadsT = 256;
constexpr float kPOffset = 15.0f;  // p <= 2^15 (below f16's largest value)

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// D += A (16 x 16, row) B (16 x 8, col), f16 in, f32 sums.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes global -> shared without passing registers; ok = false fills with zeros (src unread).
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Tile of the warp-level kernel: 8 warps = WM row groups of 16 query rows x WN.  For the scores a
// warp takes KPS / WN keys of its row group, for p V it takes HD / WN output dims over all KPS
// keys; p crosses through shared memory.  K and V stages share one ring of slots (KPS rows of
// HD + 8 halves: the 16-byte skew keeps ldmatrix free of bank conflicts).
template <int HD, int WM, bool F32>
struct Warp {
  static constexpr int WN = 8 / WM;
  static constexpr int ROWS = 16 * WM;
  static constexpr int KPS = HD == 512 ? 32 : 64;
  static constexpr int KW = KPS / WN;      // keys of a warp in the score product
  static constexpr int NKT = KW / 8;       // its 8-key columns
  static constexpr int DW = HD / WN;       // output dims of a warp
  static constexpr int PITCH = HD + 8;     // halves
  static constexpr int PPITCH = KPS + 8;
  static constexpr int TERMS = F32 ? 2 : 1;
  static constexpr int SLOT = KPS * PITCH * 2;
  static constexpr int Q_BYTES = TERMS * ROWS * PITCH * 2;
  static constexpr int P_BYTES = TERMS * ROWS * PPITCH * 2;
  static constexpr int MISC = 2 * WN * ROWS * 4 + ROWS * 4 + ROWS * 16 + 256;
  static constexpr int FIT = (227 * 1024 - Q_BYTES - P_BYTES - MISC) / SLOT;
  static constexpr int SLOTS = FIT > 8 ? 8 : FIT;
  static constexpr size_t SMEM = (size_t)Q_BYTES + P_BYTES + MISC + (size_t)SLOTS * SLOT;
  static_assert(NKT == 1 || NKT == 2 || NKT == 4, "score columns");
  static_assert(DW % 16 == 0 && SLOTS >= 3, "tile shape");
};

// Where a CTA stands in its run of stages.
struct Cursor {
  Seq s;
  int b, item, j;  // item = kv head * tiles + tile
  __device__ __forceinline__ void settle(const TreeParams& p) {  // skip what has no stages
    while (b < p.batch && (s.stages == 0 || item == p.nkh * s.tiles)) {
      item = 0;
      if (++b < p.batch) s = seq_of(p, b);
    }
  }
  __device__ __forceinline__ void next(const TreeParams& p) {
    if (++j == s.stages) {
      j = 0;
      item++;
      settle(p);
    }
  }
};

template <int HD, int WM, bool F32>
__global__ void __launch_bounds__(kThreadsT, 1) tree_warp_kernel(const TreeParams p) {
  using C = Warp<HD, WM, F32>;
  constexpr int WN = C::WN, ROWS = C::ROWS, KPS = C::KPS, NKT = C::NKT, PITCH = C::PITCH, PP = C::PPITCH;
  constexpr int NT = C::DW / 8, SLOTS = C::SLOTS;
  extern __shared__ __align__(128) unsigned char smem[];
  __half* sq = reinterpret_cast<__half*>(smem);                       // [terms][ROWS][PITCH]
  __half* sp = reinterpret_cast<__half*>(smem + C::Q_BYTES);          // [terms][ROWS][PP]
  unsigned char* misc = smem + C::Q_BYTES + C::P_BYTES;
  Sees* ssee = reinterpret_cast<Sees*>(misc);                         // [ROWS]
  float* smax = reinterpret_cast<float*>(misc + ROWS * 16);           // [WN][ROWS]
  float* ssum = smax + WN * ROWS;                                     // [WN][ROWS]
  float* sscale = ssum + WN * ROWS;                                   // [ROWS]
  unsigned char* sok = reinterpret_cast<unsigned char*>(sscale + ROWS);  // [SLOTS][8]
  unsigned char* ring = smem + C::Q_BYTES + C::P_BYTES + C::MISC;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp / WN, wn = warp % WN, g = lane >> 2, c = lane & 3;
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();

  // ---- this CTA's run of stages
  Split sp_;
  sp_.of(total_stages(p), (int)gridDim.x);
  const long long cta = blockIdx.x;
  if (cta >= sp_.active) return;
  const long long s0 = sp_.begin(cta), s1 = sp_.begin(cta + 1);
  const int n_stages = (int)(s1 - s0);
  Cursor cur;
  {
    long long first = 0;
    cur.b = find_seq(p, s0, first);
    if (cur.b >= p.batch) return;
    cur.s = seq_of(p, cur.b);
    cur.item = (int)((s0 - first) / cur.s.stages);
    cur.j = (int)((s0 - first) % cur.s.stages);
  }
  Cursor ld = cur;  // the loads run ahead

  // ---- loads: half-stage 2i is K of stage i, 2i + 1 its V.  A warp brings KPS / 8 rows; lane r
  // looks up the offset of its r-th row (K and V rows have the same one).
  constexpr int RW = KPS / 8, CH = HD / 8, RPI = CH < 32 ? 32 / CH : 1, CPL = CH > 32 ? CH / 32 : 1;
  long long off = -1;
  int loaded = 0;
  auto issue = [&](int half) {
    if (loaded < n_stages) {
      const bool is_v = half & 1;
      const int slot = half % SLOTS;
      if (!is_v) {
        off = -1;
        const int key = ld.s.lo + ld.j * KPS + warp * RW + lane;
        if (lane < RW && key < ld.s.L) off = row_offset(p, ld.b, ld.item / ld.s.tiles, key);
        const unsigned ok = __ballot_sync(0xffffffffu, off >= 0);
        if (lane == 0) sok[slot * 8 + warp] = (unsigned char)ok;
      }
      const __half* src = is_v ? p.v : p.k;
      const uint32_t dst0 = g4a::smem_u32(ring + (size_t)slot * C::SLOT);
      const int ch_real = p.hd / 8;
#pragma unroll
      for (int it = 0; it < RW / RPI; it++) {
        const int r = CH < 32 ? it * RPI + lane / CH : it;
        const long long o = __shfl_sync(0xffffffffu, off, r);
#pragma unroll
        for (int u = 0; u < CPL; u++) {
          const int ch = CH < 32 ? lane % CH : lane + 32 * u;
          const bool ok = o >= 0 && ch < ch_real;
          cp16(dst0 + (warp * RW + r) * (PITCH * 2) + ch * 16, src + (ok ? o + ch * 8 : 0), ok);
        }
      }
      if (is_v) {
        loaded++;
        if (loaded < n_stages) ld.next(p);
      }
    }
    cp_commit();  // an empty group past the end keeps the count
  };
  for (int h = 0; h < SLOTS - 1; h++) issue(h);

  float o[NT][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float sc0 = 0.f, sc1 = 0.f;
  Sees see0 = {}, see1 = {};
  int kfull = 0, j_first = 0;
  bool fresh = true;
  const int row_a = wm * 16 + g;  // this thread's rows of the tile: row_a and row_a + 8

  for (int i = 0; i < n_stages; i++) {
    cp_wait<SLOTS - 2>();
    __syncthreads();  // K of this stage is here; every warp is done with the previous V
    issue(2 * i + SLOTS - 1);

    const int kvh = cur.item / cur.s.tiles, tile = cur.item - kvh * cur.s.tiles;
    const int live = min(ROWS, cur.s.T * p.group - tile * ROWS);
    if (fresh) {
      // ---- the tile's queries and what its rows see
      j_first = cur.j;
      for (int r = warp; r < ROWS; r += 8) {
        const int gr = tile * ROWS + r, t = gr / p.group;
        const bool in = r < live;
        const size_t at = ((size_t)(cur.s.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group)) * p.hd;
        if constexpr (F32) {
          const float* src = reinterpret_cast<const float*>(p.q) + at;
          float4 x[(HD + 127) / 128];
          float big = 0.f;
#pragma unroll
          for (int u = 0; u < (HD + 127) / 128; u++) {
            const int d = (u * 32 + lane) * 4;
            x[u] = (in && d < p.hd) ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            big = fmaxf(big, fmaxf(fmaxf(fabsf(x[u].x), fabsf(x[u].y)), fmaxf(fabsf(x[u].z), fabsf(x[u].w))));
          }
#pragma unroll
          for (int w = 16; w >= 1; w >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, w));
          int e = 0;
          if (big > 0.f && big < INFINITY) e = 10 - ilogbf(big);
          e = max(-120, min(120, e));
          const float up = __int_as_float((127 + e) << 23);
          if (lane == 0) sscale[r] = ldexpf(p.scale_log2, -e);
#pragma unroll
          for (int u = 0; u < (HD + 127) / 128; u++) {
            const int d = (u * 32 + lane) * 4;
            if (d < HD) {
              const float v[4] = {x[u].x * up, x[u].y * up, x[u].z * up, x[u].w * up};
              float lo[4];
#pragma unroll
              for (int k = 0; k < 4; k++) lo[k] = v[k] - __half2float(__float2half_rn(v[k]));
              *reinterpret_cast<uint2*>(sq + r * PITCH + d) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
              *reinterpret_cast<uint2*>(sq + (ROWS + r) * PITCH + d) =
                  make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
            }
          }
        } else {
          const __half* src = reinterpret_cast<const __half*>(p.q) + at;
          if (lane == 0) sscale[r] = p.scale_log2;
          for (int d = lane * 8; d < HD; d += 256)
            *reinterpret_cast<uint4*>(sq + r * PITCH + d) =
                (in && d < p.hd) ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (lane == 0) {
          Sees v = {0, ~0ull};  // rows past the last one: their results are not written
          if (in) v = sees_of(p, cur.s, t);
          ssee[r] = v;
        }
      }
      __syncthreads();
      see0 = ssee[row_a];
      see1 = ssee[row_a + 8];
      sc0 = sscale[row_a];
      sc1 = sscale[row_a + 8];
      int km = lane < ROWS ? ssee[lane].kmin : 0;
      if (ROWS > 32) km = max(km, ssee[lane + 32].kmin);
      kfull = (int)__reduce_max_sync(0xffffffffu, (unsigned)km);
#pragma unroll
      for (int n = 0; n < NT; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
      fresh = false;
    }

    // ---- scores of 16 rows x KW keys
    const int kslot = (2 * i) % SLOTS;
    const __half* sk = reinterpret_cast<const __half*>(ring + (size_t)kslot * C::SLOT);
    constexpr int NACC = NKT == 1 ? 4 : 2;  // independent sums: hi and lo terms, odd and even steps
    float acc[NACC][NKT][4];
#pragma unroll
    for (int a = 0; a < NACC; a++)
#pragma unroll
      for (int n = 0; n < NKT; n++) acc[a][n][0] = acc[a][n][1] = acc[a][n][2] = acc[a][n][3] = 0.f;
    const uint32_t qa = g4a::smem_u32(sq + (wm * 16 + (lane & 15)) * PITCH + (lane >> 4) * 8);
    constexpr uint32_t q_lo = ROWS * PITCH * 2;
    if constexpr (NKT == 1) {
      const uint32_t ka = g4a::smem_u32(sk + (wn * 8 + (lane & 7)) * PITCH + (lane >> 3) * 8);
#pragma unroll 4
      for (int ks = 0; ks < HD / 32; ks++) {
        uint32_t kb[4], a0[4], a1[4];
        ldsm4(ka + ks * 64, kb);
        ldsm4(qa + ks * 64, a0);
        ldsm4(qa + ks * 64 + 32, a1);
        mma(acc[0][0], a0, kb[0], kb[1]);
        mma(acc[2][0], a1, kb[2], kb[3]);
        if constexpr (F32) {
          ldsm4(qa + q_lo + ks * 64, a0);
          ldsm4(qa + q_lo + ks * 64 + 32, a1);
          mma(acc[1][0], a0, kb[0], kb[1]);
          mma(acc[3][0], a1, kb[2], kb[3]);
        }
      }
    } else {
      const uint32_t ka =
          g4a::smem_u32(sk + (wn * C::KW + (lane & 7) + ((lane >> 4) & 1) * 8) * PITCH + ((lane >> 3) & 1) * 8);
#pragma unroll 4
      for (int ks = 0; ks < HD / 16; ks++) {
        uint32_t a0[4], a1[4], kb[NKT / 2][4];
        ldsm4(qa + ks * 32, a0);
        if constexpr (F32) ldsm4(qa + q_lo + ks * 32, a1);
#pragma unroll
        for (int n = 0; n < NKT / 2; n++) ldsm4(ka + n * 16 * PITCH * 2 + ks * 32, kb[n]);
        const int even = F32 ? 0 : ks & 1;
#pragma unroll
        for (int n = 0; n < NKT / 2; n++) {
          mma(acc[even][2 * n], a0, kb[n][0], kb[n][1]);
          mma(acc[even][2 * n + 1], a0, kb[n][2], kb[n][3]);
        }
        if constexpr (F32) {
#pragma unroll
          for (int n = 0; n < NKT / 2; n++) {
            mma(acc[1][2 * n], a1, kb[n][0], kb[n][1]);
            mma(acc[1][2 * n + 1], a1, kb[n][2], kb[n][3]);
          }
        }
      }
    }
    float s[NKT][4];
#pragma unroll
    for (int n = 0; n < NKT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float x = acc[0][n][e] + acc[1][n][e];
        if constexpr (NACC == 4) x += acc[2][n][e] + acc[3][n][e];
        s[n][e] = x * (e < 2 ? sc0 : sc1);
      }

    // ---- mask, running maximum
    const int key0 = cur.s.lo + cur.j * KPS;
    constexpr unsigned long long all_ok = RW == 8 ? ~0ull : 0x0f0f0f0f0f0f0f0full;
    const unsigned long long ok = *reinterpret_cast<const unsigned long long*>(sok + kslot * 8);
    const bool clean = ok == all_ok && key0 >= kfull && key0 + KPS <= cur.s.base;
    if (!clean) {
#pragma unroll
      for (int n = 0; n < NKT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int kk = wn * C::KW + n * 8 + 2 * c + (e & 1), key = key0 + kk;
          const Sees& v = e < 2 ? see0 : see1;
          bool in = (ok >> ((kk / RW) * 8 + kk % RW)) & 1;
          in = in && (key < cur.s.base ? key >= v.kmin : (v.bits >> (key - cur.s.base)) & 1);
          if (!in) s[n][e] = -INFINITY;
        }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < NKT; n++) {
      x0 = fmaxf(x0, fmaxf(s[n][0], s[n][1]));
      x1 = fmaxf(x1, fmaxf(s[n][2], s[n][3]));
    }
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
    }
    if (c == 0) {
      smax[wn * ROWS + row_a] = x0;
      smax[wn * ROWS + row_a + 8] = x1;
    }
    __syncthreads();
    float n0 = m0, n1 = m1;
#pragma unroll
    for (int w = 0; w < WN; w++) {
      n0 = fmaxf(n0, smax[w * ROWS + row_a]);
      n1 = fmaxf(n1, smax[w * ROWS + row_a + 8]);
    }
    // (a row that has seen nothing yet keeps m = -inf: its p are 2^(-inf) = 0)
    const float u0 = n0 == -INFINITY ? 0.f : n0 - kPOffset, u1 = n1 == -INFINITY ? 0.f : n1 - kPOffset;
    const float f0 = n0 == m0 ? 1.f : g4a::fast_exp2(m0 - n0), f1 = n1 == m1 ? 1.f : g4a::fast_exp2(m1 - n1);
    m0 = n0;
    m1 = n1;
    l0 *= f0;
    l1 *= f1;
    __half* pr = sp + row_a * PP + wn * C::KW + 2 * c;
#pragma unroll
    for (int n = 0; n < NKT; n++) {
      const float p0 = g4a::fast_exp2(s[n][0] - u0), p1 = g4a::fast_exp2(s[n][1] - u0);
      const float p2 = g4a::fast_exp2(s[n][2] - u1), p3 = g4a::fast_exp2(s[n][3] - u1);
      l0 += p0 + p1;
      l1 += p2 + p3;
      *reinterpret_cast<uint32_t*>(pr + n * 8) = pack2(p0, p1);
      *reinterpret_cast<uint32_t*>(pr + 8 * PP + n * 8) = pack2(p2, p3);
      if constexpr (F32) {
        *reinterpret_cast<uint32_t*>(pr + ROWS * PP + n * 8) =
            pack2(p0 - __half2float(__float2half_rn(p0)), p1 - __half2float(__float2half_rn(p1)));
        *reinterpret_cast<uint32_t*>(pr + (ROWS + 8) * PP + n * 8) =
            pack2(p2 - __half2float(__float2half_rn(p2)), p3 - __half2float(__float2half_rn(p3)));
      }
    }
    if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
        o[n][0] *= f0;
        o[n][1] *= f0;
        o[n][2] *= f1;
        o[n][3] *= f1;
      }
    }
    cp_wait<SLOTS - 2>();
    __syncthreads();  // V and p are here; every warp is done with K
    issue(2 * i + SLOTS);

    // ---- o += p V over the stage's keys
    const __half* sv = reinterpret_cast<const __half*>(ring + (size_t)((2 * i + 1) % SLOTS) * C::SLOT);
    // Where rows of the tile see different keys, a masked key's p = 0 would still turn an infinite
    // or NaN V into NaN: such a stage (rare twice over) is summed key by key over the p that are
    // not 0.
    bool bad_v = false;
    if (!clean) {
      unsigned bits = 0;
      for (int k = tid; k < KPS * HD / 8; k += kThreadsT) {
        const uint4 u = *reinterpret_cast<const uint4*>(sv + (k / CH) * PITCH + (k % CH) * 8);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++)
          bits |= ((w[e] & 0x7c00u) == 0x7c00u) | ((w[e] & 0x7c000000u) == 0x7c000000u);
      }
      bad_v = __syncthreads_or((int)bits);
    }
    if (bad_v) {
      for (int k = 0; k < KPS; k++) {
        float pa = __half2float(sp[row_a * PP + k]), pb = __half2float(sp[(row_a + 8) * PP + k]);
        if constexpr (F32) {
          pa += __half2float(sp[(ROWS + row_a) * PP + k]);
          pb += __half2float(sp[(ROWS + row_a + 8) * PP + k]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(sv + k * PITCH + wn * C::DW + n * 8 + 2 * c));
          if (pa != 0.f) o[n][0] = fmaf(pa, v.x, o[n][0]), o[n][1] = fmaf(pa, v.y, o[n][1]);
          if (pb != 0.f) o[n][2] = fmaf(pb, v.x, o[n][2]), o[n][3] = fmaf(pb, v.y, o[n][3]);
        }
      }
    } else {
      const uint32_t pa = g4a::smem_u32(sp + (wm * 16 + (lane & 15)) * PP + (lane >> 4) * 8);
      const uint32_t va =
          g4a::smem_u32(sv + ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + wn * C::DW + (lane >> 4) * 8);
#pragma unroll
      for (int ks = 0; ks < KPS / 16; ks++) {
        uint32_t a0[4], a1[4];
        ldsm4(pa + ks * 32, a0);
        if constexpr (F32) ldsm4(pa + ROWS * PP * 2 + ks * 32, a1);
#pragma unroll
        for (int n = 0; n < NT / 2; n++) {
          uint32_t vb[4];
          ldsm4t(va + ks * 16 * PITCH * 2 + n * 32, vb);
          mma(o[2 * n], a0, vb[0], vb[1]);
          mma(o[2 * n + 1], a0, vb[2], vb[3]);
          if constexpr (F32) {
            mma(o[2 * n], a1, vb[0], vb[1]);
            mma(o[2 * n + 1], a1, vb[2], vb[3]);
          }
        }
      }
    }

    // ---- end of the tile's stages in this CTA
    if (cur.j + 1 == cur.s.stages || i + 1 == n_stages) {
#pragma unroll
      for (int w = 1; w <= 2; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
      }
      if (c == 0) {
        ssum[wn * ROWS + row_a] = l0;
        ssum[wn * ROWS + row_a + 8] = l1;
      }
      __syncthreads();
      l0 = l1 = 0.f;
#pragma unroll
      for (int w = 0; w < WN; w++) {
        l0 += ssum[w * ROWS + row_a];
        l1 += ssum[w * ROWS + row_a + 8];
      }
      const bool whole = j_first == 0 && cur.j + 1 == cur.s.stages;
      if (whole) {
        // (l is NaN, not 0, for a row with a NaN score)
        const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = row_a + 8 * h;
          if (r >= live) continue;
          const int gr = tile * ROWS + r, t = gr / p.group;
          const size_t at = ((size_t)(cur.s.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group)) * p.hd;
          const float inv = h ? i1 : i0;
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const int d = wn * C::DW + n * 8 + 2 * c;
            if (d >= p.hd) continue;
            const float y0 = o[n][2 * h] * inv, y1 = o[n][2 * h + 1] * inv;
            if constexpr (F32)
              *reinterpret_cast<float2*>(reinterpret_cast<float*>(p.out) + at + d) = make_float2(y0, y1);
            else
              *reinterpret_cast<uint32_t*>(reinterpret_cast<__half*>(p.out) + at + d) = pack2(y0, y1);
          }
        }
      } else {
        // slot 0: the tile with which this CTA's run begins; slot 1: one that starts later in it
        const bool later = i - (cur.j - j_first) > 0;
        float* part = p.part + (size_t)(2 * cta + (later ? 1 : 0)) * ROWS * (HD + 2);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = row_a + 8 * h;
#pragma unroll
          for (int n = 0; n < NT; n++)
            *reinterpret_cast<float2*>(part + (size_t)r * HD + wn * C::DW + n * 8 + 2 * c) =
                make_float2(o[n][2 * h], o[n][2 * h + 1]);
          if (wn == 0 && c == 0) {
            part[ROWS * HD + r] = h ? m1 : m0;
            part[ROWS * HD + ROWS + r] = h ? l1 : l0;
          }
        }
      }
      fresh = true;
    }
    if (i + 1 < n_stages) cur.next(p);
  }
}

// Joins the parts of every tile that was cut between CTAs, one CTA per (cut, query row): cut x is
// the border between the runs of CTA x and x + 1.  If it lies inside a tile and is the first that
// does, the tile's parts are in slot 1 of the CTA that began it (slot 0 if that CTA's run begins
// with the tile) and slot 0 of the following ones.
template <bool F32>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeParams p) {
  __shared__ float red[8];
  __shared__ float4 sum[128];
  const int tid = threadIdx.x, lane = tid & 31;
  g4a::pdl_wait_primary();
  g4a::pdl_launch_dependents();
  Split sp;
  sp.of(total_stages(p), p.grid);
  const long long cut = (long long)blockIdx.x + 1;
  if (cut >= sp.active) return;
  const long long s = sp.begin(cut);
  long long first = 0;
  const int b = find_seq(p, s, first);
  if (b >= p.batch) return;
  const Seq q = seq_of(p, b);
  const int item = (int)((s - first) / q.stages);
  const long long a = first + (long long)item * q.stages;  // the tile's first stage
  if (s == a || sp.begin(cut - 1) > a) return;              // not inside, or not the first inside
  const int kvh = item / q.tiles, tile = item - kvh * q.tiles;
  const int gr = tile * p.rows + (int)blockIdx.y, t = gr / p.group;
  if (t >= q.T) return;
  const long long c0 = cut - 1, c1 = sp.owner(a + q.stages - 1);
  const int n = (int)(c1 - c0) + 1;
  const size_t stride = (size_t)p.rows * (p.hd_pad + 2);
  auto slot = [&](int i) { return p.part + (size_t)(2 * (c0 + i) + (i == 0 && a > sp.begin(c0) ? 1 : 0)) * stride; };
  // the largest m, then the weights and the sum of l
  float m = -INFINITY;
  for (int i = tid; i < n; i += 128) m = fmaxf(m, __ldcg(slot(i) + (size_t)p.rows * p.hd_pad + blockIdx.y));
#pragma unroll
  for (int w = 16; w >= 1; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  if (lane == 0) red[tid >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  // 16-byte columns of the row x lanes over the parts
  const int cols = p.hd_pad / 4, lanes = 128 / (cols < 128 ? cols : 128), col = tid % cols, pl = tid / cols;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int i = pl; i < n; i += lanes) {
    const float* base = slot(i);
    const float mi = __ldcg(base + (size_t)p.rows * p.hd_pad + blockIdx.y);
    const float li = __ldcg(base + (size_t)p.rows * p.hd_pad + p.rows + blockIdx.y);
    const float4 x = __ldcg(reinterpret_cast<const float4*>(base + (size_t)blockIdx.y * p.hd_pad) + col);
    const float w = mi == -INFINITY ? 0.f : g4a::fast_exp2(mi - m);
    if (mi == -INFINITY && li == 0.f) continue;  // saw nothing
    l = fmaf(w, li, l);
    o.x = fmaf(w, x.x, o.x);
    o.y = fmaf(w, x.y, o.y);
    o.z = fmaf(w, x.z, o.z);
    o.w = fmaf(w, x.w, o.w);
  }
  sum[tid] = o;
  __syncthreads();
  if (col == 0) red[pl] = l;
  __syncthreads();
  if (pl == 0 && col * 4 < p.hd) {
    float lt = 0.f;
    for (int i = 0; i < lanes; i++) lt += red[i];
    for (int i = 1; i < lanes; i++) {
      const float4 x = sum[i * cols + col];
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    const size_t at = ((size_t)(q.row0 + t) * p.nqh + kvh * p.group + (gr - t * p.group)) * p.hd + col * 4;
    if constexpr (F32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
      *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + at) =
          make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    }
  }
}

template <int HD, int WM, bool F32>
g4a_status launch_warp(g4a_ctx* ctx, TreeParams& p, long long stages_upper_keys, long long tiles_upper) {
  using C = Warp<HD, WM, F32>;
  static std::atomic<bool> done[64];
  if (ctx->device >= 64 || !done[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(tree_warp_kernel<HD, WM, F32>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(tree_warp_kernel)");
    if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
  }
  p.rows = C::ROWS;
  p.kps = C::KPS;
  p.hd_pad = HD;
  const long long stages = stages_upper_keys / C::KPS + tiles_upper;
  p.grid = (int)std::max<long long>(1, std::min<long long>(stages, ctx->num_sms));
  if (g4a_status s = g4a_ensure_workspace(ctx, (size_t)2 * p.grid * C::ROWS * (HD + 2) * sizeof(float))) return s;
  p.part = static_cast<float*>(ctx->workspace);
  {
    g4a_prof_scope ps(ctx, G4A_PROF_TREE_ATTN);
    const cudaError_t e =
        g4a_launch(tree_warp_kernel<HD, WM, F32>, dim3(p.grid), dim3(kThreadsT), C::SMEM, ctx->stream, true, p);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch tree_warp_kernel");
  }
  if (p.grid > 1) {
    g4a_prof_scope ps(ctx, G4A_PROF_TREE_MERGE);
    const cudaError_t e = g4a_launch(tree_merge_kernel<F32>, dim3(p.grid - 1, C::ROWS), dim3(128), 0, ctx->stream,
                                     true, p);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch tree_merge_kernel");
  }
  return G4A_OK;
}

template <bool F32>
g4a_status dispatch_warp(g4a_ctx* ctx, TreeParams& p, const int32_t* host_kv_lens, uint64_t cap) {
  // tile height: 64 rows, or 32 where a kv head has no more (and at head_dim 512, where a
  // 64-row tile does not fit)
  const int rows_max = p.max_tokens * p.group;
  const int rows = (p.hd > 256 || rows_max <= 32) ? 32 : 64;
  const long long tiles = (rows_max + rows - 1) / rows;
  long long keys = 0;
  for (int b = 0; b < p.batch; b++) {
    uint64_t L = host_kv_lens ? (uint64_t)(host_kv_lens[b] < 0 ? 0 : host_kv_lens[b]) : cap;
    if (L > cap) L = cap;
    if (p.window != 0u && L > (uint64_t)p.window + p.max_tokens) L = (uint64_t)p.window + p.max_tokens;
    keys += (long long)L;
  }
  keys *= tiles * p.nkh;
  const long long items = tiles * p.nkh * p.batch;
  if (p.hd > 256) return launch_warp<512, 2, F32>(ctx, p, keys, items);
  if (p.hd > 128)
    return rows == 32 ? launch_warp<256, 2, F32>(ctx, p, keys, items) : launch_warp<256, 4, F32>(ctx, p, keys, items);
  if (p.hd > 64)
    return rows == 32 ? launch_warp<128, 2, F32>(ctx, p, keys, items) : launch_warp<128, 4, F32>(ctx, p, keys, items);
  return rows == 32 ? launch_warp<64, 2, F32>(ctx, p, keys, items) : launch_warp<64, 4, F32>(ctx, p, keys, items);
}

}  // namespace

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
    return g4a_fail(G4A_EINVAL, "%s: max_tokens %u not in [1, %d] (longer prompts: g4a_prefill_attn)", fn, max_tokens,
                    kMaxTokens);
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
  return format == G4A_ACT_F32 ? dispatch_warp<true>(ctx, p, host_kv_lens, cap)
                               : dispatch_warp<false>(ctx, p, host_kv_lens, cap);
}
