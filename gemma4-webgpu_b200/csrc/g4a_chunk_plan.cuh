// How the work of g4a_chunk_attn_paged is dealt out: tiles, key blocks, and the pieces that chunk_plan_kernel
// writes for the attention kernel and the join.
#pragma once

#include "g4a_chunk.cuh"

namespace g4a_chunk {

constexpr int kTileRows = 256;  // query rows of a tile: (token, q head of the group), both CTAs of a pair together
constexpr int kMaxPairs = 128;
constexpr int kPlanThreads = 1024;
// Stages that a piece costs besides its keys: queries, the first scores and softmax without an MMA beside them,
// epilogue.
constexpr int kLead = 3;
// And the join, if any tile is cut: ns for itself, and bytes per ns that it (and the writing) takes for the parts.
constexpr float kJoinNs = 3500.f, kJoinRate = 2500.f;

// A run of a tile's key blocks for one pair of CTAs.
struct Piece {
  int b, head;      // sequence; kv head * (halves of the head dims) + half
  int tile;         // rows tile * 256 ..
  int j0, j1;       // its stages, of all those of the tile
  int slot;         // where its partial result goes; -1: the whole tile, straight to the output
  int row0, T, L;   // the sequence
  int sinks, skip;  // stages [0, sinks) are blocks [0, sinks), stage j behind them is block j + skip
  int pad;
};

// A tile that several pieces share: the first's result is in `slot`, the others' in slot1, slot1 + step, ...
struct Cut {
  int b, head, tile, row0, T, parts, slot, slot1, step;
  __device__ __forceinline__ int slot_of(int part) const { return part == 0 ? slot : slot1 + (part - 1) * step; }
};

struct Plan {
  int cuts, pad[3];
  int4 pair[kMaxPairs];  // x, x + z, ... below y: the pieces of each pair
};

// What the planning kernel reads and writes besides ChunkParams.
struct PlanParams {
  ChunkParams c;
  int pairs, halves, kb_log2;  // halves of the head dims; keys of a block (masses: of a tile)
  int max_slots;
  long long max_entries;  // tiles that there is room for (more: the sequences' rows of q overlap)
  float stage_bytes, stage_ns;  // of a block: what is loaded, about how long it takes
  float part_bytes;             // of a whole tile's partial result
  int block_tokens, head_chunks;  // masses: tokens of a row block, row blocks for the heads of one token
  Plan* plan;
  Piece* pieces;
  Cut* cuts;
  int4* seqs;          // [batch + 1]: tile entries before, items before, most stages of a tile, (chunks) pieces before
  long long* entries;  // [tile entries]: stages of all earlier entries
  int2* parts;         // masses: [items] the pair of a tile's first piece, number of its pieces
};

// (num_tokens * num_q_heads is below 2^31, so rows of a kv head, and of a tile past them, are numbers of 32 bits)
__device__ __forceinline__ int tiles_of(const ChunkParams& p, const Seq& s) {
  return (int)(((uint32_t)s.T * (uint32_t)p.group + kTileRows - 1) / kTileRows);
}
__device__ __forceinline__ int first_token(const ChunkParams& p, int tile) {
  return (int)((uint32_t)tile * kTileRows / (uint32_t)p.group);
}
__device__ __forceinline__ int last_token(const ChunkParams& p, int T, int tile) {
  return (int)min((uint32_t)T - 1u, ((uint32_t)(tile + 1) * kTileRows - 1u) / (uint32_t)p.group);
}

// The key blocks that a tile's rows see: [0, sinks) and [window0, window1).
struct Blocks {
  int sinks, window0, window1;
  __device__ __forceinline__ int count() const { return sinks + window1 - window0; }
};
__device__ __forceinline__ Blocks blocks_of(const ChunkParams& p, const Seq& s, int tile, int kb_log2) {
  const int lo = first_in_window(p, s.base() + first_token(p, tile)), hi = s.base() + last_token(p, s.T, tile) + 1;
  const int up = (1 << kb_log2) - 1;
  Blocks r;
  r.window0 = lo >> kb_log2;
  r.window1 = (hi + up) >> kb_log2;
  r.sinks = (int)((min((long long)p.sinks, (long long)lo) + up) >> kb_log2);
  if (r.sinks >= r.window0) r.sinks = r.window0 = 0;  // they meet
  return r;
}

// Masses: the key tiles that any token of a sequence sees, as the blocks of one tile that holds all tokens.
__device__ __forceinline__ Blocks key_tiles_of(const ChunkParams& p, const Seq& s, int kb_log2) {
  Blocks r = {0, 0, 0};
  if (s.T <= 0) return r;
  const int lo = first_in_window(p, s.base()), up = (1 << kb_log2) - 1;
  r.window0 = lo >> kb_log2;
  r.window1 = (int)(((long long)s.L + up) >> kb_log2);
  r.sinks = (int)((min((long long)p.sinks, (long long)lo) + up) >> kb_log2);
  if (r.sinks >= r.window0) r.sinks = r.window0 = 0;
  return r;
}
// The tokens [first, last) that see any key of the tile at k0.
struct Tokens {
  int first, last;
};
__device__ __forceinline__ Tokens tokens_of(const ChunkParams& p, const Seq& s, int k0, int keys) {
  Tokens t = {max(0, k0 - s.base()), s.T};
  if (p.window != 0u && (uint32_t)k0 >= p.sinks)
    t.last = (int)min((long long)s.T, (long long)k0 + keys - 1 + (long long)p.window - s.base());
  return t;
}

}  // namespace g4a_chunk
cudaError_t g4a_chunk_plan_launch(g4a_ctx* ctx, const g4a_chunk::PlanParams& a, bool masses, long long entries);
