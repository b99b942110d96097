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
  int rows, kps;  // query rows of a tile, keys of a stage (of the launched kernel)
  int grid;       // CTAs of the launched kernel
  float* part;    // [2 * grid] partial rows: o [rows, hd_pad] | m [rows] | l [rows]
  int hd_pad;
  struct Cut* cuts;  // [2 * grid]
  const __half* q_terms;  // f32 queries: [tokens, nqh][2][hd_pad], high and low f16 terms
  const float* q_scale;   // and [tokens, nqh] scale * log2(e) over the power of two in them
  int* err;
};

// A tile whose keys were not all done by one CTA, written by the CTA that has its first piece, at the
// index of that piece's slot.
struct Cut {
  int parts;             // pieces (chunks == 1) or chunks to be joined; 0: nothing
  int rows;              // query rows of the tile that exist
  int row0;              // the sequence's first row of q
  int kvh, first;        // kv head; the tile's first row in units of (token, head of the group)
  int stages, chunks, tiles, tile;
  int each, extra;       // the split of the list over the CTAs
  long long base;        // stage of the list at which the (sequence, kv head) begins
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
  s.tiles = (s.T * p.group + p.rows - 1) / p.rows;
  s.stages = s.tiles > 0 ? (L - s.lo + p.kps - 1) / p.kps : 0;
  return s;
}

__device__ __forceinline__ long long stages_of(const TreeParams& p, const Seq& s) {
  return (long long)p.nkh * s.tiles * s.stages;
}

// The list of all stages is cut into equal runs, one per CTA; only the first min(grid, total) CTAs
// have work.  Order: sequence, kv head, chunk of keys, tile, stage.  The tiles of a kv head read the
// same keys, so its keys are cut into chunks about as long as a run and a chunk's tiles follow one
// another: their CTAs read the same rows at the same time, and only the first reads them from HBM.
// (Tile after tile, the six tiles of a 131,000-key context came past each row 90 MB apart and the L2
// had lost it.)  A chunk is at least as long as a run, so a run holds at most two pieces of tiles
// that are not whole: one that begins before or with it and one that goes on after it.
// Division of non-negative numbers that are nearly always below 2^32 (the 64-bit one is a long
// sequence, and the walk starts with several of them).
__device__ __forceinline__ long long quot(long long a, long long b) {
  if ((((unsigned long long)a | (unsigned long long)b) >> 32) == 0) return (long long)((uint32_t)a / (uint32_t)b);
  return a / b;
}

struct Split {
  long long total, active, each, extra;
  __device__ __forceinline__ void of(long long t, int grid) {
    total = t;
    active = grid < t ? grid : t;
    each = active ? quot(t, active) : 0;
    extra = t - each * active;
  }
  __device__ __forceinline__ long long begin(long long c) const { return c * each + (c < extra ? c : extra); }
  // the CTA whose run holds stage s
  __device__ __forceinline__ long long owner(long long s) const {
    const long long cut = extra * (each + 1);
    return s < cut ? quot(s, each + 1) : extra + quot(s - cut, each);
  }
};

// First stage of chunk c of n stages in `chunks`.
__device__ __forceinline__ int chunk_at(int n, int chunks, int c) { return (int)quot((long long)n * c, chunks); }

// Where a role stands in the CTA's run of stages.
struct Walk {
  Seq s;
  int b, kvh, tile;
  int chunks, chunk, j, j_end;  // stage of the tile; end of the chunk

  __device__ __forceinline__ void chunk_of(const Split& split) {
    chunks = s.tiles > 1 ? max(1, (int)quot(s.stages, max(1ll, split.each))) : 1;
  }
  // stage `local` of sequence b's list
  __device__ __forceinline__ void seek(const TreeParams& p, const Split& split, int seq, long long local) {
    b = seq;
    s = seq_of(p, b);
    chunk_of(split);
    const long long per_head = (long long)s.tiles * s.stages;
    kvh = (int)quot(local, per_head);
    local -= kvh * per_head;
    chunk = (int)quot(quot(local, s.tiles) * chunks, s.stages);
    while (chunk > 0 && local < (long long)s.tiles * chunk_at(s.stages, chunks, chunk)) chunk--;
    while (local >= (long long)s.tiles * chunk_at(s.stages, chunks, chunk + 1)) chunk++;
    const int j0 = chunk_at(s.stages, chunks, chunk);
    j_end = chunk_at(s.stages, chunks, chunk + 1);
    local -= (long long)s.tiles * j0;
    tile = (int)quot(local, j_end - j0);
    j = j0 + (int)(local - (long long)tile * (j_end - j0));
  }
  // past the end of a tile's chunk
  __device__ __forceinline__ void next_piece(const TreeParams& p, const Split& split) {
    if (++tile == s.tiles) {
      tile = 0;
      if (++chunk == chunks) {
        chunk = 0;
        if (++kvh == p.nkh) {
          kvh = 0;
          do {
            if (++b >= p.batch) {
              s.stages = 0;
              return;
            }
            s = seq_of(p, b);
          } while (s.stages == 0);
          chunk_of(split);
        }
      }
    }
    j = chunk_at(s.stages, chunks, chunk);
    j_end = chunk_at(s.stages, chunks, chunk + 1);
  }
  __device__ __forceinline__ void next(const TreeParams& p, const Split& split) {
    if (++j == j_end) next_piece(p, split);
  }
  __device__ __forceinline__ bool begins() const { return j == chunk_at(s.stages, chunks, chunk); }
  // the first key from which every row sees all of the prefix
  __device__ __forceinline__ int kfull(const TreeParams& p) const {
    const long long k = p.window ? (long long)s.base + s.T - (long long)p.window : 0;
    return k < 0 ? 0 : k > s.base ? s.base : (int)k;
  }
  __device__ __forceinline__ int key0(const TreeParams& p) const { return s.lo + j * p.kps; }
  __device__ __forceinline__ bool clean(const TreeParams& p) const {
    return key0(p) >= kfull(p) && key0(p) + p.kps <= s.base;
  }
};

// Total stages over the batch, by one full warp (every lane returns it).
__device__ __forceinline__ long long total_stages(const TreeParams& p) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) n += stages_of(p, seq_of(p, b));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// The sequence that holds flattened stage s (s < total) and the first stage of that sequence; one
// full warp, every lane returns them.
__device__ __forceinline__ int find_seq(const TreeParams& p, long long s, long long& first) {
  const int lane = threadIdx.x & 31;
  long long acc = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const long long n = b < p.batch ? stages_of(p, seq_of(p, b)) : 0;
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const long long start = acc + incl - n;
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && s >= start && s < start + n);
    if (hit) {
      const int src = __ffs(hit) - 1;
      first = __shfl_sync(0xffffffffu, start, src);
      return b0 + src;
    }
    acc += __shfl_sync(0xffffffffu, incl, 31);
  }
  first = acc;
  return p.batch;
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
