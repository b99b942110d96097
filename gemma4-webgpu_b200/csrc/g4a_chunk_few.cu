// g4a_chunk_attn_paged for few query rows to a sequence (decode steps): mma.sync straight from global memory.
//
// Eight query rows are a fraction of a tcgen05 tile, and a decode step is bound by the HBM, so here nothing is staged:
// a warp takes 16 keys at a time, and a lane loads 16 consecutive bytes of K or V rows and uses them as MMA operands
// as they are.
//   S [rows x 8 keys] = Q K^T   m16n8k16, A = Q (rows 8-15 are zeros), B = K: lane 4 g + t has dims 32 s + 8 t .. + 7 of
//                               key g; the order of the dims in the product is free, so those are its operands.
//   O^T [16 dims x rows] += V^T P^T   A = V^T: lane 4 g + t has 8 dims of the keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, and
//                               pairs up two keys' values of a dim by one byte permute; the 16 dims of a product are
//                               dim i of eight lanes' pieces in two 64-dim chunks.  B = P^T: what the first product
//                               leaves in a lane (row g, keys 2 t, 2 t + 1) is the operand that the second one wants.
// A warp has 16 KB under way (K and V of 16 keys, 256 dims), an SM 128 KB, more than the HBM's latency needs.  Heads of
// more than 256 dims: two warps share 16 keys, half of the dims each, and add up their halves of the scores.
// The sequences' keys are dealt to the CTAs in equal parts, as many CTAs as the SMs hold at once, but no sequence gets more
// than four times its share of the CTAs (the partial results have places by that; one sequence of 131,000 rows takes 46 us,
// with 63 of 500 beside it, which leave it 20 CTAs, 232); the warps of a CTA meet in shared memory, the parts of a row tile
// in a second kernel.  Softmax as in the tcgen05 kernel: m follows the
// maximum lazily, p rounded to f16 for the product with V and summed unrounded.
// 64 decode sequences of up to 12,000 rows of 256 dims: 106 us, 5.0 TB/s; one token over 512 rows of a window: 10.6 us,
// the two kernels' latency.  Fetching the next step into the L2 ahead made the first 309 us.
#include <float.h>

#include <algorithm>
#include <atomic>

#include "g4a_chunk.cuh"

namespace {

using namespace g4a;
using namespace g4a_chunk;

constexpr int kWarps = 4, kStepKeys = 16, kTile = 8;  // warps of a CTA; keys of a step; query rows of a tile
constexpr int kNoKey = -1 - 0x7fffffff;
constexpr float kRaiseF = 15.0f, kBelowF = 3.0f, kUnseenF = -FLT_MAX;  // (of m, as in the tcgen05 kernel)

struct FewParams {
  ChunkParams c;
  int splits;   // CTAs of a sequence and kv head, at most
  int ctas;     // CTAs to be dealt out; 0 (more sequences than threads): every sequence has `splits` of them
  float* part;  // [row tiles][nkh][splits] (o [8][hd] | m [8] | l [8])
};

// The steps of 16 keys that a row tile sees, [0, sinks) and [w0, w1), and how many CTAs share them.
struct Steps {
  int sinks, w0, w1, parts;
  __device__ __forceinline__ int count() const { return sinks + w1 - w0; }
};
__device__ __forceinline__ Steps steps_of(const FewParams& a, const Seq& s, int tile, int groups, int parts) {
  const ChunkParams& p = a.c;
  const int t0 = (int)((uint32_t)(tile * kTile) / (uint32_t)p.group);
  const int t1 = min(s.T - 1, (int)((uint32_t)(tile * kTile + kTile - 1) / (uint32_t)p.group));
  const int lo = first_in_window(p, s.base() + t0), hi = s.base() + t1 + 1;
  Steps r;
  r.w0 = lo / kStepKeys;
  r.w1 = (hi + kStepKeys - 1) / kStepKeys;
  r.sinks = (int)((min((long long)p.sinks, (long long)lo) + kStepKeys - 1) / kStepKeys);
  if (r.sinks >= r.w0) r.sinks = r.w0 = 0;
  r.parts = min(parts, (r.count() + groups - 1) / groups);  // a step for each of a CTA's groups at least
  return r;
}
// The steps that thread b's sequence is dealt out by.
__device__ __forceinline__ int steps_to_deal(const ChunkParams& p) {
  if ((int)threadIdx.x >= p.batch) return 0;
  const Seq s = seq_of(p, (int)threadIdx.x, (long long)p.max_pages * p.page_size);
  if (s.T <= 0) return 0;
  const int lo = first_in_window(p, s.base());
  return (int)((min((long long)p.sinks, (long long)lo) + kStepKeys - 1) / kStepKeys) + (s.L + kStepKeys - 1) / kStepKeys -
         lo / kStepKeys;
}
// Place of a row tile among all of the call's (a sequence has T group / 8 + 1 at most).
__device__ __forceinline__ size_t tile_place(const ChunkParams& p, const Seq& s, int b, int tile) {
  return (size_t)((uint32_t)((long long)s.row0 * p.group / kTile)) + (size_t)b + (size_t)tile;
}

__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Sets infinite and NaN halves to 0; whether there was one.
__device__ __forceinline__ bool clear_bad(uint32_t& w) {
  const uint32_t was = w;
  if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
  if ((w & 0x7c000000u) == 0x7c000000u) w &= 0x0000ffffu;
  return w != was;
}

// SEG: 32-dim segments of a warp's share of a head; SHARE: warps that share a head's dims.  Three CTAs to an SM where the
// registers allow (64 ragged sequences of 128 dims 54 us, with two 63; with four, which spill, 66).
template <int SEG, int SHARE>
__global__ void __launch_bounds__(kWarps * 32, SEG > 4 ? 2 : 3) chunk_few_kernel(const FewParams a) {
  constexpr int DIMS = SEG * 32, CH = DIMS / 64, GROUPS = kWarps / SHARE;
  constexpr int PITCH = DIMS + 4;  // floats from row to row where the warps meet
  const ChunkParams& p = a.c;
  __shared__ __align__(16) uint4 q_s[SHARE][SEG][32];  // Q as operands: [segment][lane]
  __shared__ float s_s[SHARE > 1 ? kWarps : 1][4][32];  // halves of the scores
  __shared__ float m_s[kWarps][kTile], l_s[kWarps][kTile];
  extern __shared__ __align__(16) float o_s[];  // [warps][8 rows][PITCH]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int share = warp % SHARE, group = warp / SHARE;
  int b = (int)(blockIdx.y / (unsigned)p.nkh), kvh = (int)(blockIdx.y % (unsigned)p.nkh), split = (int)blockIdx.x, most = a.splits;
  pdl_wait_primary();
  pdl_launch_dependents();
  if (a.ctas > 0) {
    const Deal d = deal_out<kWarps * 32>(steps_to_deal(p), p.nkh, a.ctas, a.splits, GROUPS, (int)blockIdx.x, -1);
    if (d.b < 0) return;
    b = d.b, kvh = d.local / d.parts, split = d.local - kvh * d.parts, most = d.parts;
  }
  const Seq s = seq_of(p, b, (long long)p.max_pages * p.page_size);
  const int base = s.base(), rows = s.T * p.group, d_warp = share * DIMS;
  const int* table = p.page_table + (size_t)b * p.max_pages;
  for (int tile = 0; tile * kTile < rows; tile++) {
    const Steps st = steps_of(a, s, tile, GROUPS, most);
    if (split >= st.parts) continue;
    const int n = st.count(), i0 = (int)((long long)n * split / st.parts), i1 = (int)((long long)n * (split + 1) / st.parts);
    // row g of the tile (rows that are not there: the last token's sight, no weight in anything that is kept)
    const int r = min(tile * kTile + g, rows - 1), token = (int)((uint32_t)r / (uint32_t)p.group);
    const int pos = base + token, lo = first_in_window(p, pos);
    const int pos0 = base + (int)((uint32_t)(tile * kTile) / (uint32_t)p.group);  // of the tile's first row
    const int pos1 = base + (int)((uint32_t)min(tile * kTile + kTile - 1, rows - 1) / (uint32_t)p.group);
    const int lo0 = first_in_window(p, pos0), lo1 = first_in_window(p, pos1);
    if (group == 0) {
      const bool live = tile * kTile + g < rows;
      const __half* row = p.q + ((size_t)(s.row0 + token) * p.nqh + (size_t)kvh * p.group + (r - token * p.group)) * p.hd;
#pragma unroll
      for (int e = 0; e < SEG; e++) {
        const int d = d_warp + e * 32 + t * 8;
        q_s[share][e][lane] = live && d < p.hd ? *reinterpret_cast<const uint4*>(row + d) : make_uint4(0, 0, 0, 0);
      }
    }
    __syncthreads();
    float m = kUnseenF, l = 0.f, o[CH / 2][8][4];
#pragma unroll
    for (int c = 0; c < CH / 2; c++)
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[c][i][k] = 0.f;
    bool taken = false;  // values of V that are not finite
    // The page of key g (+ 8) of a step, looked up one step ahead; -1: nobody sees the key
    auto first_key = [&](int i) { return (i < st.sinks ? i : i - st.sinks + st.w0) * kStepKeys; };
    auto page_of = [&](int i, int h) {
      const int key = first_key(i) + g + 8 * h;
      return i < i1 && key <= pos1 && (key >= lo0 || (uint32_t)key < p.sinks) ? table[(uint32_t)key / (uint32_t)p.page_size] : kNoKey;
    };
    int pages[2] = {page_of(i0 + group, 0), page_of(i0 + group, 1)};
    for (int i = i0 + group; i < i1; i += GROUPS) {
      const int k0 = first_key(i);
      // where this lane's rows of K (keys g, g + 8) and V (2 t, 2 t + 1, 2 t + 8, 2 t + 9) lie; -1: not there
      long long at_k[2], at_v[4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t key = (uint32_t)(k0 + g + 8 * h);
        at_k[h] = (((long long)pages[h] * p.page_size + key % (uint32_t)p.page_size) * p.nkh + kvh) * p.hd + d_warp;
        if (pages[h] < 0 || pages[h] >= p.num_pages) {
          if (pages[h] != kNoKey) atomicExch(p.err, G4A_DEVERR_PAGE);
          at_k[h] = -1;
        }
      }
#pragma unroll
      for (int h = 0; h < 4; h++)  // (a lane of the same key has looked it up: key 2 t + h is row 2 t + h of K, and so on)
        at_v[h] = __shfl_sync(0xffffffffu, h < 2 ? at_k[0] : at_k[1], (2 * t + (h & 1)) * 4);
      uint4 k[2][SEG], v[4][CH];
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < SEG; e++)
          k[h][e] = at_k[h] >= 0 && d_warp + e * 32 + t * 8 < p.hd
                        ? load_once(p.k + at_k[h] + e * 32 + t * 8)
                        : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int h = 0; h < 4; h++)
#pragma unroll
        for (int c = 0; c < CH; c++)
          v[h][c] = at_v[h] >= 0 && d_warp + c * 64 + g * 8 < p.hd
                        ? load_once(p.v + at_v[h] + c * 64 + g * 8)
                        : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int h = 0; h < 2; h++) pages[h] = page_of(i + GROUPS, h);
      float x[4];  // row g, keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < SEG; e++) {
          const uint4 q = q_s[share][e][lane];
          mma_16x8x16(c, q.x, 0u, q.y, 0u, k[h][e].x, k[h][e].y);
          mma_16x8x16(c, q.z, 0u, q.w, 0u, k[h][e].z, k[h][e].w);
        }
        x[2 * h] = c[0];
        x[2 * h + 1] = c[1];
      }
      if constexpr (SHARE > 1) {
#pragma unroll
        for (int h = 0; h < 4; h++) s_s[warp][h][lane] = x[h];
        named_bar_sync(1 + group, SHARE * 32);  // (both warps take the same steps)
#pragma unroll
        for (int h = 0; h < 4; h++) x[h] = s_s[group * SHARE][h][lane] + s_s[group * SHARE + 1][h][lane];
        named_bar_sync(1 + group, SHARE * 32);
      }
      const bool clean = k0 + kStepKeys <= pos0 + 1 && (k0 >= lo1 || (uint32_t)(k0 + kStepKeys) <= p.sinks);
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const int key = k0 + 2 * t + (h & 1) + (h >> 1) * 8;
        x[h] *= p.scale_log2;
        if (at_v[h] < 0 || (!clean && !(key <= pos && (key >= lo || (uint32_t)key < p.sinks)))) x[h] = -INFINITY;
        top = fmaxf(top, x[h]);
      }
      if (!clean) {  // 0 x inf is NaN: what is not finite is taken out and added at the end for the rows that see it
#pragma unroll
        for (int h = 0; h < 4; h++)
#pragma unroll
          for (int c = 0; c < CH; c++) {
            taken |= clear_bad(v[h][c].x);
            taken |= clear_bad(v[h][c].y);
            taken |= clear_bad(v[h][c].z);
            taken |= clear_bad(v[h][c].w);
          }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool raise = top > m + kRaiseF;
      if (__any_sync(0xffffffffu, raise)) {
        const float m_new = raise ? top - kBelowF : m;
        const float fall = raise ? (m == kUnseenF ? 0.f : fast_exp2(m - m_new)) : 1.f;
        l *= fall;
        m = m_new;
        const float f0 = __shfl_sync(0xffffffffu, fall, 8 * t), f1 = __shfl_sync(0xffffffffu, fall, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < CH / 2; c++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            o[c][e][0] *= f0;
            o[c][e][1] *= f1;
            o[c][e][2] *= f0;
            o[c][e][3] *= f1;
          }
      }
      float w[4];
#pragma unroll
      for (int h = 0; h < 4; h++) w[h] = fast_exp2(x[h] - m);
      l += (w[0] + w[1]) + (w[2] + w[3]);
      const uint32_t b0 = half2_of(w[0], w[1]), b1 = half2_of(w[2], w[3]);
#pragma unroll
      for (int c = 0; c < CH / 2; c++) {
        auto word = [&](int h, int ch, int e) {
          const uint4& u = v[h][ch];
          return e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
        };
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t pick = (e & 1) ? 0x7632u : 0x5410u;  // the upper or the lower halves
          mma_16x8x16(o[c][e], __byte_perm(word(0, 2 * c, e), word(1, 2 * c, e), pick),
              __byte_perm(word(0, 2 * c + 1, e), word(1, 2 * c + 1, e), pick),
              __byte_perm(word(2, 2 * c, e), word(3, 2 * c, e), pick),
              __byte_perm(word(2, 2 * c + 1, e), word(3, 2 * c + 1, e), pick), b0, b1);
        }
      }
    }
    // ---- the warps meet
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) m_s[warp][g] = m, l_s[warp][g] = l;
    float* mine = o_s + (size_t)warp * kTile * PITCH;
#pragma unroll
    for (int c = 0; c < CH / 2; c++)
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int k = 0; k < 4; k++)  // row 2 t + (k & 1), dim 8 g + e of chunk 2 c + (k >> 1)
          mine[(2 * t + (k & 1)) * PITCH + (2 * c + (k >> 1)) * 64 + 8 * g + e] = o[c][e][k];
    taken = __syncthreads_or(taken);
    for (int row = warp; row < kTile; row += kWarps) {  // of the tile
      float mx = kUnseenF, lt = 0.f;
#pragma unroll
      for (int i = 0; i < GROUPS; i++) mx = fmaxf(mx, m_s[i * SHARE][row]);
      float f[GROUPS];
#pragma unroll
      for (int i = 0; i < GROUPS; i++) {
        f[i] = m_s[i * SHARE][row] == mx ? 1.f : fast_exp2(m_s[i * SHARE][row] - mx);
        lt = fmaf(f[i], l_s[i * SHARE][row], lt);
      }
      const int gr = tile * kTile + row;
      if (gr < rows) {
        const int tok = (int)((uint32_t)gr / (uint32_t)p.group);
        const size_t out_row = (size_t)(s.row0 + tok) * p.nqh + (size_t)kvh * p.group + (gr - tok * p.group);
        float* part = a.part + ((tile_place(p, s, b, tile) * p.nkh + kvh) * a.splits + split) * (size_t)(kTile * (p.hd + 2));
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        for (int d = lane * 4; d < p.hd; d += 128) {
          const int of = d / DIMS, in = d - of * DIMS;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int i = 0; i < GROUPS; i++) {
            const float4 u = *reinterpret_cast<const float4*>(o_s + ((size_t)(i * SHARE + of) * kTile + row) * PITCH + in);
            y.x = fmaf(f[i], u.x, y.x);
            y.y = fmaf(f[i], u.y, y.y);
            y.z = fmaf(f[i], u.z, y.z);
            y.w = fmaf(f[i], u.w, y.w);
          }
          if (taken) {  // (rare) the values that were taken out of this part's steps, for the keys that the row sees
            const int p_row = base + tok;
            for (int i = i0; i < i1; i++) {
              const int k0 = first_key(i);
              if (k0 + kStepKeys <= pos0 + 1 && (k0 >= lo1 || (uint32_t)(k0 + kStepKeys) <= p.sinks)) continue;
              for (int key = k0; key < k0 + kStepKeys && key <= p_row; key++) {
                if (!sees(p, p_row, key)) continue;
                const long long at = row_offset(p, b, kvh, key);
                if (at < 0) continue;
                float* const to[4] = {&y.x, &y.y, &y.z, &y.w};
                for (int c = 0; c < 4; c++) {
                  const float z = __half2float(p.v[at + d + c]);
                  if (!(fabsf(z) < INFINITY)) *to[c] += z;
                }
              }
            }
          }
          if (st.parts == 1)
            *reinterpret_cast<uint2*>(p.out + out_row * p.hd + d) =
                make_uint2(half2_of(y.x * inv, y.y * inv), half2_of(y.z * inv, y.w * inv));
          else
            *reinterpret_cast<float4*>(part + (size_t)row * p.hd + d) = y;
        }
        if (lane == 0) {
          if (st.parts == 1) {
            if (p.lse != nullptr) p.lse[out_row] = lt == 0.f ? -INFINITY : (mx + log2f(lt)) * kLn2C;
          } else {
            part[(size_t)kTile * p.hd + row] = mx;
            part[(size_t)kTile * p.hd + kTile + row] = lt;
          }
        }
      }
    }
    __syncthreads();
  }
}

// Joins a row tile's parts: a CTA has 8 rows x 32 dims, 8 float4 of a row in 8 lanes, and 4 threads for each that share
// the parts.
__global__ void __launch_bounds__(256) chunk_few_join_kernel(const FewParams a, int groups) {
  const ChunkParams& p = a.c;
  __shared__ float4 so[4][64];
  __shared__ float sm[4][8], sl[4][8];
  const int b = (int)(blockIdx.y / (unsigned)p.nkh), kvh = (int)(blockIdx.y % (unsigned)p.nkh);
  const int c = threadIdx.x & 7, row = (threadIdx.x >> 3) & 7, lanes = threadIdx.x >> 6, d = (int)blockIdx.x * 32 + c * 4;
  pdl_wait_primary();
  pdl_launch_dependents();
  const int most = a.ctas > 0 ? deal_out<256>(steps_to_deal(p), p.nkh, a.ctas, a.splits, groups, 0, b).parts : a.splits;
  const Seq s = seq_of(p, b, (long long)p.max_pages * p.page_size);
  const int rows = s.T * p.group;
  for (int tile = 0; tile * kTile < rows; tile++) {
    const int parts = steps_of(a, s, tile, groups, most).parts;
    if (parts == 1) continue;
    const size_t pitch = (size_t)kTile * (p.hd + 2);
    const float* part = a.part + (tile_place(p, s, b, tile) * p.nkh + kvh) * a.splits * pitch;
    const bool live = tile * kTile + row < rows && d < p.hd;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      constexpr int kFly = 8;
      for (int i0 = lanes; i0 < parts; i0 += 4 * kFly) {
        float mi[kFly], li[kFly];
        float4 x[kFly];
#pragma unroll
        for (int f = 0; f < kFly; f++) {
          const int i = i0 + 4 * f;
          mi[f] = -INFINITY, li[f] = 0.f, x[f] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i >= parts) continue;
          const float* at = part + i * pitch;
          mi[f] = __ldcg(at + (size_t)kTile * p.hd + row);
          li[f] = __ldcg(at + (size_t)kTile * p.hd + kTile + row);
          x[f] = __ldcg(reinterpret_cast<const float4*>(at + (size_t)row * p.hd + d));
        }
        float mn = m;
#pragma unroll
        for (int f = 0; f < kFly; f++) mn = fmaxf(mn, mi[f]);
        const float wo = m == mn ? 1.f : fast_exp2(m - mn);
        m = mn;
        l *= wo;
        o.x *= wo, o.y *= wo, o.z *= wo, o.w *= wo;
#pragma unroll
        for (int f = 0; f < kFly; f++) {
          const float wf = mi[f] == mn ? 1.f : fast_exp2(mi[f] - mn);
          l = fmaf(wf, li[f], l);
          o.x = fmaf(wf, x[f].x, o.x);
          o.y = fmaf(wf, x[f].y, o.y);
          o.z = fmaf(wf, x[f].z, o.z);
          o.w = fmaf(wf, x[f].w, o.w);
        }
      }
    }
    if (c == 0) sm[lanes][row] = m, sl[lanes][row] = l;
    so[lanes][threadIdx.x & 63] = o;
    __syncthreads();
    if (lanes == 0 && live) {
      float mx = m;
      for (int i = 1; i < 4; i++) mx = fmaxf(mx, sm[i][row]);
      l = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < 4; i++) {
        const float wf = sm[i][row] == mx ? 1.f : fast_exp2(sm[i][row] - mx);
        const float4 x = so[i][threadIdx.x];
        l = fmaf(wf, sl[i][row], l);
        o.x = fmaf(wf, x.x, o.x);
        o.y = fmaf(wf, x.y, o.y);
        o.z = fmaf(wf, x.z, o.z);
        o.w = fmaf(wf, x.w, o.w);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int gr = tile * kTile + row, tok = (int)((uint32_t)gr / (uint32_t)p.group);
      const size_t to = (size_t)(s.row0 + tok) * p.nqh + (size_t)kvh * p.group + (gr - tok * p.group);
      *reinterpret_cast<uint2*>(p.out + to * p.hd + d) =
          make_uint2(half2_of(o.x * inv, o.y * inv), half2_of(o.z * inv, o.w * inv));
      if (p.lse != nullptr && d == 0) p.lse[to] = l == 0.f ? -INFINITY : (mx + log2f(l)) * kLn2C;
    }
    __syncthreads();
  }
}

template <int SEG, int SHARE>
g4a_status launch(g4a_ctx* ctx, const ChunkParams& p) {
  constexpr int groups = kWarps / SHARE;
  constexpr size_t smem = (size_t)kWarps * kTile * (SEG * 32 + 4) * sizeof(float);
  static std::atomic<bool> ready[64];
  if (ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(chunk_few_kernel<SEG, SHARE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "cudaFuncSetAttribute(chunk_few_kernel)");
    if (ctx->device < 64) ready[ctx->device].store(true, std::memory_order_release);
  }
  FewParams a = {};
  a.c = p;
  const long long heads = (long long)p.batch * p.nkh;
  // rows that a sequence can read, in CTAs with a step for every group
  const uint64_t cap = (uint64_t)p.page_size * p.max_pages;
  uint64_t keys = cap;
  if (p.window != 0u) keys = std::min<uint64_t>(cap, (uint64_t)p.window + p.sinks + 4 * kStepKeys);
  const long long most = (long long)((keys + groups * kStepKeys - 1) / (groups * kStepKeys));
  // One round of CTAs, equal parts, while the heads are few: half a round more than the heads at least, or the parts are
  // too uneven.  With more heads there have to be more parts than CTAs at once:
  //  - up to 128 dims four to a head from half a round on (64 ragged sequences x 4 heads 155 us, one round 181; x 8
  //    heads 269, two to a head 286; as many equal ones 103 and 121, 198 and 237);
  //  - above, two to a head from a round on (64 ragged sequences x 8 heads 322 us, one round 351), not before (x 4 heads
  //    324 us, two to a head 355, though 50 x 4 heads 303 and 289).
  // A sequence has four times its share at most.
  const long long room = (SEG > 4 ? 2ll : 3ll) * ctx->num_sms;
  const bool many = SEG > 4 ? heads >= room : 2 * heads >= room;
  const long long ctas = many ? (SEG > 4 ? 2 : 4) * heads : std::max(room, heads + room / 2);
  if (p.batch <= kWarps * 32) {
    a.ctas = (int)std::min(ctas, heads * most + heads);
    a.splits = (int)std::min(most, 4 * ((ctas + heads - 1) / heads));
  } else {
    a.splits = (int)std::max<long long>(1, std::min(most, (3 * ctas + heads - 1) / heads));
  }
  const size_t tiles = (size_t)((long long)p.tokens * p.group / kTile) + (size_t)p.batch;
  const size_t need = tiles * p.nkh * a.splits * kTile * (p.hd + 2) * sizeof(float);
  if (g4a_status s = g4a_ensure_workspace(ctx, need)) return s;
  a.part = static_cast<float*>(ctx->workspace);
  g4a_prof_scope ps(ctx, G4A_PROF_CHUNK_ATTN);
  cudaError_t e = g4a_launch(chunk_few_kernel<SEG, SHARE>, a.ctas > 0 ? dim3((unsigned)a.ctas) : dim3((unsigned)a.splits, (unsigned)heads), dim3(kWarps * 32), smem,
                             ctx->stream, true, a);
  if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_few_kernel");
  if (a.splits > 1) {
    e = g4a_launch(chunk_few_join_kernel, dim3((unsigned)((p.hd + 31) / 32), (unsigned)heads), dim3(256), 0, ctx->stream,
                   true, a, groups);
    if (e != cudaSuccess) return g4a_cuda_fail(e, "launch chunk_few_join_kernel");
  }
  return G4A_OK;
}

}  // namespace

g4a_status g4a_chunk_few_launch(g4a_ctx* ctx, const ChunkParams& p) {
  if (p.hd > 256) return launch<8, 2>(ctx, p);
  if (p.hd > 128) return launch<8, 1>(ctx, p);
  return launch<4, 1>(ctx, p);
}
