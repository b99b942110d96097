// What the kernels of g4a_tree_attn_paged share: the work partition and the visibility rules.
#pragma once

#include "g4a_internal.cuh"

namespace g4a_tree {

constexpr int kMaxTokens = 64;  // drafted tokens of a sequence (bits of a tree mask)
constexpr float kLog2eT = 1.4426950408889634f;

struct TreeParams {
  const void* q;  // [tokens, nqh, hd] f32 or f16
  void* out;
  const __half *k, *v;  // page pools [num_pages, page_size, nkh, hd]
  const int *page_table, *kv_lens, *q_indptr;
  const unsigned long long* mask;  // per token, or null (chain)
  int tokens, batch, max_tokens;
  int page_size, max_pages, num_pages;
  int nqh, nkh, group, hd;  // group = nqh / nkh
  float scale_log2;         // scale * log2(e)
  uint32_t window;
  int rows_log2;  // query rows of a tile of the launched kernel, 2^rows_log2
  int grid;       // CTAs of the launched kernel
  float* part;    // [2 * grid] partial rows: o [rows, hd_pad] | m [rows] | l [rows]
  int hd_pad;
  struct Cut* cuts;  // [2 * grid]
  const __half* q_terms;  // f32 queries: [tokens, nqh][2][hd_pad], high and low f16 terms
  const float* q_scale;   // and [tokens, nqh] scale * log2(e) over the power of two in them
  int* err;
};

constexpr int kStageLog2 = 7;  // keys of a stage: 128

// A tile whose keys were not all done by one CTA, written by the CTA that has its first piece, at the
// index of that piece's slot k; the other pieces are in slots (k & ~1) + i * stride.
struct Cut {
  int parts;       // pieces; 0: nothing
  int stride;
  int rows;        // query rows of the tile that exist
  int row0;        // the sequence's first row of q
  int kvh, first;  // kv head; the tile's first row in units of (token, head of the group)
};

// One sequence: T drafted tokens (rows row0 .. of q), base older rows, keys [lo, L) to be read.
// T = 0: nothing to do (also for a sequence that does not fit together, which is reported).
struct Seq {
  int row0, T, base, L, lo;
  int tiles;   // query tiles of one kv head
  int stages;  // key stages of one tile
};

__device__ __forceinline__ Seq seq_of(const TreeParams& p, int b) {
  Seq s = {};
  const int r0 = p.q_indptr[b], r1 = p.q_indptr[b + 1], L = p.kv_lens[b];
  const long long cap = (long long)p.max_pages * p.page_size;
  if (r0 < 0 || r1 < r0 || r1 > p.tokens || r1 - r0 > p.max_tokens || L < r1 - r0 || L > cap) {
    atomicExch(p.err, G4A_DEVERR_TREE);
    return s;
  }
  s.row0 = r0;
  s.T = r1 - r0;
  s.L = L;
  s.base = L - s.T;
  // the earliest key any token's window can reach (a token that sees itself alone: base + 1 - W;
  // one whose mask is empty: base - W)
  s.lo = (p.window != 0u && (uint32_t)s.base > p.window) ? s.base - (int)p.window : 0;
  s.tiles = (s.T * p.group + (1 << p.rows_log2) - 1) >> p.rows_log2;
  s.stages = s.tiles > 0 ? (L - s.lo + (1 << kStageLog2) - 1) >> kStageLog2 : 0;
  return s;
}

__device__ __forceinline__ long long stages_of(const TreeParams& p, const Seq& s) {
  return (long long)p.nkh * s.tiles * s.stages;
}

// Division of non-negative numbers that are nearly always below 2^32 (the 64-bit one is a long
// sequence of instructions).
__device__ __forceinline__ long long quot(long long a, long long b) {
  if ((((unsigned long long)a | (unsigned long long)b) >> 32) == 0) return (long long)((uint32_t)a / (uint32_t)b);
  return a / b;
}

// First stage of chunk c of n stages in `chunks`; the first n % chunks have one more.
__device__ __forceinline__ int chunk_at(int n, int chunks, int c) {
  const uint32_t part = (uint32_t)n / (uint32_t)chunks, rest = (uint32_t)n - part * (uint32_t)chunks;
  return (int)(part * (uint32_t)c + min((uint32_t)c, rest));
}

// How the tiles' stages are dealt to the CTAs, found by every warp for itself from the lengths on the
// device.
//  - One piece per CTA (`run` > 0), where that costs little balance: each kv head's keys are cut into
//    the fewest chunks of at most `run` stages, run the smallest length found for which the pieces
//    (chunk, tile) are no more than the CTAs, and CTA c does piece c, in the order sequence, kv head,
//    chunk, tile.  A chunk's tiles are neighbours and read the same rows at the same time, so only
//    one of them goes to HBM.  (Tile after tile, the six tiles of a 131,000-key context came past
//    each row 90 MB apart and the L2 had lost it: 321 us instead of 221.)  A piece's start and end
//    cost as much as two to four stages, so one longer piece beats two (64 tokens over 32k keys: 78
//    -> 64 us) unless the longest is more than a quarter (and a stage) above the mean.
//  - Else the list of all stages (sequence, kv head, tile, stage) is cut into equal runs, where a tile
//    counts `lead` stages more than it has, in front: its queries, join and epilogue.  A run holds whole
//    tiles, and at most two pieces: one at its begin, one at its end.
struct Plan {
  int run, lead;
  long long active, each, extra;
  long long origin;  // where the tile begins in which this CTA's run begins, in the list with the leads
  __device__ __forceinline__ long long begin(long long c) const { return c * each + (c < extra ? c : extra); }
  // the CTA whose run holds stage s
  __device__ __forceinline__ long long owner(long long s) const {
    const long long cut = extra * (each + 1);
    return s < cut ? quot(s, each + 1) : extra + quot(s - cut, each);
  }
};

// Where a role stands in the CTA's stages.
struct Walk {
  Seq s;
  int b, kvh, tile;
  int chunks, chunk, j, j_end;  // stage of the tile; end of the chunk

  // past the last stage of a tile (more tiles than CTAs: one chunk)
  __device__ __forceinline__ void next_tile(const TreeParams& p) {
    j = 0;
    if (++tile < s.tiles) return;
    tile = 0;
    if (++kvh < p.nkh) return;
    kvh = 0;
    do {
      if (++b >= p.batch) {
        s.stages = j_end = 0;
        return;
      }
      s = seq_of(p, b);
    } while (s.stages == 0);
    j_end = s.stages;
  }
  // the first key from which every row sees all of the prefix
  __device__ __forceinline__ int kfull(const TreeParams& p) const {
    const long long k = p.window ? (long long)s.base + s.T - (long long)p.window : 0;
    return k < 0 ? 0 : k > s.base ? s.base : (int)k;
  }
  __device__ __forceinline__ int key0() const { return s.lo + (j << kStageLog2); }
  __device__ __forceinline__ bool clean(const TreeParams& p) const {
    return key0() >= kfull(p) && key0() + (1 << kStageLog2) <= s.base;
  }
};

__device__ __forceinline__ void seek_piece(const TreeParams& p, int run, int b, const Seq& s, uint32_t local, Walk& at) {
  at.s = s;
  at.b = b;
  at.chunks = (int)((uint32_t)(s.stages + run - 1) / (uint32_t)run);
  const uint32_t q = local / (uint32_t)s.tiles;
  at.tile = (int)(local - q * (uint32_t)s.tiles);
  at.kvh = (int)(q / (uint32_t)at.chunks);
  at.chunk = (int)(q - (uint32_t)at.kvh * (uint32_t)at.chunks);
  at.j = chunk_at(s.stages, at.chunks, at.chunk);
  at.j_end = chunk_at(s.stages, at.chunks, at.chunk + 1);
}
__device__ __forceinline__ void seek_stage(const TreeParams& p, int b, const Seq& s, long long local, Walk& at) {
  at.s = s;
  at.b = b;
  const long long item = quot(local, s.stages);
  at.j = (int)(local - item * s.stages);
  at.j_end = s.stages;
  at.kvh = (int)quot(item, s.tiles);
  at.tile = (int)(item - (long long)at.kvh * s.tiles);
  at.chunks = 1;
  at.chunk = 0;
}
// Whether pieces of `run` stages are worth it where equal runs have `mean`.
__device__ __forceinline__ bool run_fits(long long run, long long mean) { return run <= mean + mean / 4 + 1; }

// The general case of deal(): any batch, totals beyond 32 bits.
static __device__ __noinline__ int deal_any(const TreeParams& p, int cta, int grid, Plan& plan, Walk& at) {
  const int lane = threadIdx.x & 31;
  auto warp_sum = [](long long n) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  };
  long long tiles = 0, total = 0;
  int longest = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const Seq s = seq_of(p, b);
    tiles += (long long)p.nkh * s.tiles;
    total += (long long)p.nkh * s.tiles * s.stages;
    longest = max(longest, s.stages);
  }
  tiles = warp_sum(tiles);
  total = warp_sum(total);
  longest = (int)__reduce_max_sync(0xffffffffu, (unsigned)longest);
  plan.run = plan.lead = 0;
  plan.active = plan.each = plan.extra = plan.origin = 0;
  if (total == 0) return 0;
  const long long mean = quot(total + grid - 1, grid);
  if (tiles <= grid) {
    long long run = min((long long)longest, mean), pieces = 0;
    for (int k = 0; k < 12; k++) {
      pieces = 0;
      for (int b = lane; b < p.batch; b += 32) {
        const Seq s = seq_of(p, b);
        pieces += (long long)p.nkh * s.tiles * quot(s.stages + run - 1, run);
      }
      pieces = warp_sum(pieces);
      if (pieces <= grid || !run_fits(run, mean)) break;
      run = min((long long)longest, max(run + 1, quot(run * pieces + grid - 1, grid)));
    }
    if (pieces <= grid && run_fits(run, mean)) {
      plan.run = (int)run;
      plan.active = pieces;
    }
  }
  if (plan.run == 0) {
    plan.active = grid < total ? grid : total;
    plan.each = quot(total, plan.active);
    plan.extra = total - plan.each * plan.active;
  }
  if (cta >= plan.active) return 0;
  const long long want = plan.run > 0 ? cta : plan.begin(cta);
  long long before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const Seq s = b0 + lane < p.batch ? seq_of(p, b0 + lane) : Seq{};
    const long long n =
        (long long)p.nkh * s.tiles * (plan.run > 0 ? quot(s.stages + plan.run - 1, plan.run) : (long long)s.stages);
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const long long start = before + incl - n;
    const unsigned found = __ballot_sync(0xffffffffu, n > 0 && want >= start && want < start + n);
    if (found) {
      const int src = __ffs(found) - 1;
      const long long local = want - __shfl_sync(0xffffffffu, start, src);
      const Seq hit = seq_of(p, b0 + src);
      if (plan.run > 0) {
        seek_piece(p, plan.run, b0 + src, hit, (uint32_t)local, at);
        return at.j_end - at.j;
      }
      seek_stage(p, b0 + src, hit, local, at);
      plan.origin = want - at.j;
      return (int)(plan.begin(cta + 1) - want);
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return 0;
}

constexpr int kTable = 512;  // sequences that deal() finds in the lanes and in shared memory
// Stages that a tile's queries, join and epilogue cost (0 / 2: 40 trees of up to 24 tokens 99 / 95 us, 32
// chains with 32-bit queries 50.6 / 48.9, 100 short sequences 37.4 / 35.9; 1 and 3 within a microsecond of 2).
constexpr int kLead = 2;

// The table's entry of sequence b: tiles of all kv heads, stages of a tile.
__device__ __forceinline__ int2 table_entry(const TreeParams& p, int b) {
  const Seq s = seq_of(p, b);
  return make_int2(p.nkh * s.tiles, s.stages);
}

// One full warp: the plan, CTA `cta`'s first stage, and their number (0: no work).  A lane holds the entry
// `own` of sequence `lane`; those from 32 on, up to kTable, lie in `table` (filled by the whole CTA: one round
// of loads).  32 bits and little code: the kernels start cold, and every line of code on this path is
// fetched before the first key is.
__device__ __forceinline__ int deal(const TreeParams& p, const int2 own, const int2* table, int cta, int grid, Plan& plan,
                                    Walk& at) {
  const int lane = threadIdx.x & 31;
  int tiles = own.x, total = own.x * own.y;
  bool large = p.batch > kTable || __umulhi((uint32_t)own.x, (uint32_t)own.y) != 0 || (uint32_t)total > 0x1fffffu;
#pragma unroll 1
  for (int b = lane + 32; b < p.batch && !large; b += 32) {
    const int2 e = table[b];
    const long long n = (long long)e.x * e.y;
    large = n > 0x1fffff;  // (kTable of these stay below 2^30)
    tiles += e.x;
    total += (int)n;
  }
  if (__any_sync(0xffffffffu, large)) return deal_any(p, cta, grid, plan, at);
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  total = __reduce_add_sync(0xffffffffu, total);
  plan.run = plan.lead = 0;
  plan.active = plan.each = plan.extra = plan.origin = 0;
  if (total == 0) return 0;
  const int mean = (int)((uint32_t)(total + grid - 1) / (uint32_t)grid);
  if (tiles <= grid) {
    int run = mean;
#pragma unroll 1
    do {
      int pieces = own.x * (int)((uint32_t)(own.y + run - 1) / (uint32_t)run);
#pragma unroll 1
      for (int b = lane + 32; b < p.batch; b += 32) {
        const int2 e = table[b];
        pieces += e.x * (int)((uint32_t)(e.y + run - 1) / (uint32_t)run);
      }
      pieces = __reduce_add_sync(0xffffffffu, pieces);
      if (pieces <= grid) {
        plan.run = run;
        plan.active = pieces;
        break;
      }
      run = max(run + 1, (int)((uint32_t)(run * pieces) / (uint32_t)grid));
    } while (run_fits(run, mean));
  }
  if (plan.run == 0) {
    plan.lead = kLead;
    total += tiles * kLead;
    plan.active = min(grid, total);
    plan.each = (uint32_t)total / (uint32_t)plan.active;
    plan.extra = total - plan.each * plan.active;
  }
  if (cta >= plan.active) return 0;
  // a run's end, then its begin (or the piece)
  int n_stages = 0;
#pragma unroll 1
  for (int k = plan.run > 0 ? 1 : 0; k < 2; k++) {
    const int want = plan.run > 0 ? cta : (int)plan.begin(cta + 1 - k);
    int before = 0, tiles_before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int2 e = b0 == 0 ? own : b0 + lane < p.batch ? table[b0 + lane] : make_int2(0, 0);
      const int n =
          e.x * (plan.run > 0 ? (int)((uint32_t)(e.y + plan.run - 1) / (uint32_t)plan.run) : e.y + plan.lead);
      int incl = n, incl_tiles = e.x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o), u = __shfl_up_sync(0xffffffffu, incl_tiles, o);
        if (lane >= o) incl += t, incl_tiles += u;
      }
      const int start = before + incl - n, tile0 = tiles_before + incl_tiles - e.x;
      // (the end of the last run lies behind the last sequence)
      const unsigned found = __ballot_sync(0xffffffffu, n > 0 && want >= start && want < start + n);
      if (found) {
        const int src = __ffs(found) - 1;
        const int local = want - __shfl_sync(0xffffffffu, start, src);
        if (plan.run > 0) {
          seek_piece(p, plan.run, b0 + src, seq_of(p, b0 + src), (uint32_t)local, at);
          return at.j_end - at.j;
        }
        const int stages = __shfl_sync(0xffffffffu, e.y, src), per = stages + plan.lead;
        const int item = (int)((uint32_t)local / (uint32_t)per), off = local - item * per;
        // stages before this place: all that is before it without the leads
        const int here = want - off - (__shfl_sync(0xffffffffu, tile0, src) + item) * plan.lead + max(0, off - plan.lead);
        if (k == 0) {
          n_stages = here;
        } else {
          n_stages -= here;
          if (n_stages > 0) seek_stage(p, b0 + src, seq_of(p, b0 + src), item * stages + max(0, off - plan.lead), at);
          plan.origin = want - off;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      tiles_before += __shfl_sync(0xffffffffu, incl_tiles, 31);
      if (k == 0 && b0 + 32 >= p.batch) n_stages = before - tiles_before * plan.lead;  // all
    }
  }
  return n_stages;
}

// Two floats rounded to an f16 pair.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What query row r of a tile's sequence sees: prefix rows [kmin, base) and the drafted rows of
// `bits`.  Of the base + popcount(mask) rows in its list only the last W stay.
struct Sees {
  int kmin;
  unsigned long long bits;
};
__device__ __forceinline__ Sees sees_of(const TreeParams& p, const Seq& s, int token) {
  const unsigned long long all = s.T >= 64 ? ~0ull : (1ull << s.T) - 1ull;
  unsigned long long m = p.mask ? p.mask[s.row0 + token] & all : (token >= 63 ? ~0ull : (2ull << token) - 1ull);
  Sees v = {0, m};
  if (p.window != 0u) {
    const int n = s.base + __popcll(m);
    int drop = (uint32_t)n > p.window ? n - (int)p.window : 0;  // of the list's first rows
    v.kmin = drop < s.base ? drop : s.base;
    for (drop -= v.kmin; drop > 0; drop--) m &= m - 1;
    v.bits = m;
  }
  return v;
}

// Element offset of cache row `key` of sequence b and kv head kvh, or -1 for a bad page id.
__device__ __forceinline__ long long row_offset(const TreeParams& p, int b, int kvh, int key) {
  const int j = key / p.page_size;
  const int page = p.page_table[(size_t)b * p.max_pages + j];
  if (page < 0 || page >= p.num_pages) {
    atomicExch(p.err, G4A_DEVERR_PAGE);
    return -1;
  }
  return (((long long)page * p.page_size + (key - j * p.page_size)) * p.nkh + kvh) * p.hd;
}

}  // namespace g4a_tree
