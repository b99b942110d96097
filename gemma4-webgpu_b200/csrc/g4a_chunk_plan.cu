// The planning kernel of g4a_chunk_attn_paged and g4a_paged_key_mass: one CTA reads the lengths on the device (so a
// captured graph follows them) and deals the work to the pairs of CTAs that the next kernel runs.
//
// An item is a tile of one kv head (of one half of its dims, where a head has two); it has as many stages as key
// blocks.  Two ways to deal them, the cheaper one by a count of stages is taken:
//  - Runs: the list of all items (sequence, kv head, tile), each kLead stages longer than it is, is cut into
//    equal runs, one for each pair.  Perfect balance; a pair has whole tiles and at most two ends of cut ones.
//  - Chunks: every tile of a sequence is cut into the same number of chunks, and the pairs take the pieces (kv head,
//    chunk, tile) in that order.  Neighbours read the same rows at the same time, so that of several tiles only
//    one goes to HBM where the L2 does not hold a sequence's rows (the runs pass a row at 16 different times in 512
//    tokens x 8 heads over 131,000 rows); and with one chunk nothing has to be joined.
// The masses turn it round: a tile is 256 keys of one kv head, its stages are blocks of the query rows that see any of
// them, and they are dealt in runs.
#include "g4a_chunk_plan.cuh"

namespace {

using namespace g4a;
using namespace g4a_chunk;

// Inclusive sums over the block's threads of N values at once; returns the totals in `all`.
template <int N>
__device__ __forceinline__ void block_scan(long long (&x)[N], long long (&all)[N], long long (*warp_sum)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; i++) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, x[i], o);
      if (lane >= o) x[i] += t;
    }
    if (lane == 31) warp_sum[warp][i] = x[i];
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      long long t = warp_sum[lane][i];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      warp_sum[lane][i] = t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (warp > 0) x[i] += warp_sum[warp - 1][i];
    all[i] = warp_sum[kPlanThreads / 32 - 1][i];
  }
  __syncthreads();
}

// The last sequence b with seqs[b].x (entries) or .y (items) <= i, of n sequences.
__device__ __forceinline__ int find_seq(const int4* seqs, int n, int i, bool items) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((items ? seqs[mid].y : seqs[mid].x) <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Division of non-negative numbers that are nearly always below 2^32 (the 64-bit one is a long sequence of instructions).
__device__ __noinline__ long long quot_wide(long long a, long long b) { return a / b; }
__device__ __forceinline__ long long quot(long long a, long long b) {
  if ((((unsigned long long)a | (unsigned long long)b) >> 32) == 0) return (long long)((uint32_t)a / (uint32_t)b);
  return quot_wide(a, b);
}

// The pieces of item i of a list that is cut into equal runs: it has n stages, and the list is `length` long, kLead for
// each item in front of its stages; this one begins at `at`.  Run w is [w length / pairs, (w + 1) length / pairs).  A
// piece of pair w lies at i + w in the list of pieces, so a pair's lie together (with holes between the pairs).  A pair
// has at most one piece that goes on from the pair before (its result in place 2 w) and one that the next goes on with
// (2 w + 1).
template <bool MASS>
__device__ __forceinline__ void emit_runs(const PlanParams& a, const Seq& s, int b, int head, int tile, const Blocks& k,
                                          int i, int items, long long at, long long n, long long length, int pairs,
                                          int* cut_count) {
  auto begin = [&](int w) { return quot((long long)w * length, pairs); };
  auto owner = [&](long long x) { return (int)quot((x + 1) * pairs - 1, length); };
  const int w0 = owner(at + kLead), parts = owner(at + kLead + n - 1) - w0 + 1;
  const int before = i > 0 ? owner(at - 1) : -1, after = i + 1 < items ? owner(at + n + 2 * kLead) : pairs;
  for (int c = 0; c < parts; c++) {
    const int w = w0 + c;
    Piece d;
    d.b = b, d.head = head, d.tile = tile, d.row0 = s.row0, d.T = s.T, d.L = s.L;
    d.j0 = c == 0 ? 0 : (int)(begin(w) - at - kLead);
    d.j1 = c == parts - 1 ? (int)n : (int)(begin(w + 1) - at - kLead);
    d.slot = parts == 1 ? -1 : c == 0 ? 2 * w + 1 : 2 * w;
    d.sinks = k.sinks, d.skip = k.window0 - k.sinks, d.pad = 0;
    a.pieces[i + w] = d;
    if (c > 0 || before < w) a.plan->pair[w].x = i + w;
    if (c < parts - 1 || after > w) a.plan->pair[w].y = i + w + 1;
  }
  if (MASS) a.parts[i] = make_int2(w0, parts);
  else if (parts > 1)
    a.cuts[atomicAdd(cut_count, 1)] = Cut{b, head, tile, s.row0, s.T, parts, 2 * w0 + 1, 2 * (w0 + 1), 2};
}

// A small call: up to kPlanThreads sequences and as many tiles, one to a thread, all in shared memory.
template <bool MASS>
__global__ void __launch_bounds__(kPlanThreads) chunk_plan_small_kernel(const PlanParams a) {
  __shared__ int warp_sum[33], row0_s[kPlanThreads], T_s[kPlanThreads], L_s[kPlanThreads], entry_s[kPlanThreads + 1];
  __shared__ int most_s[kPlanThreads], stage_s[kPlanThreads + 1], place_s[kPlanThreads];
  __shared__ float costs[32], seen_s[32];
  __shared__ int cut_count, longest_s;
  const ChunkParams& p = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long cap = MASS ? min((long long)p.max_pages * p.page_size, p.mass_stride) : (long long)p.max_pages * p.page_size;
  const int heads = p.nkh * a.halves;
  auto key_tile = [&](const Blocks& k, int e) { return e < k.sinks ? e : e + k.window0 - k.sinks; };
  // exclusive sum of x over the threads; the total in warp_sum[32]
  auto scan = [&](int x) {
    int incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      const int mine = warp_sum[lane];
      int t = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      warp_sum[lane] = t - mine;
      if (lane == 31) warp_sum[32] = t;
    }
    __syncthreads();
    return incl - x + warp_sum[warp];
  };
  if (tid == 0) cut_count = 0, longest_s = 0;
  most_s[tid] = 0;
  pdl_wait_primary();
  pdl_launch_dependents();
  // ---- sequences
  Seq mine = {0, 0, 0};
  int tiles = 0;
  float seen = 0.f;
  if (tid < p.batch) {
    mine = seq_of(p, tid, cap);
    if (mine.T > 0) {
      tiles = MASS ? key_tiles_of(p, mine, a.kb_log2).count() : tiles_of(p, mine);
      seen = (float)(mine.L - first_in_window(p, mine.base()));
    }
    row0_s[tid] = mine.row0, T_s[tid] = mine.T, L_s[tid] = mine.L;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) seen += __shfl_xor_sync(0xffffffffu, seen, o);
  if (lane == 0) seen_s[warp] = seen;
  entry_s[tid] = scan(tiles);
  const int entries = warp_sum[32], items = entries * heads;
  if (tid == 0) entry_s[kPlanThreads] = entries;
  for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
  if (MASS && tid <= p.batch) a.seqs[tid] = make_int4(0, (tid < p.batch && tid < kPlanThreads ? entry_s[tid] : entries) * heads, 0, 0);
  __syncthreads();
  if (items == 0 || entries > a.max_entries) {
    if (tid == 0) a.plan->cuts = 0;
    if (tid == 0 && items != 0) atomicExch(p.err, G4A_DEVERR_TREE);
    if (MASS && tid < p.batch) a.seqs[tid] = make_int4(0, -1, 0, 0);
    return;
  }
  // ---- tiles: a thread's sequence is the last one whose entries begin at or before it (those without any share a begin)
  int b = 0, e = 0, n = 0, tile = 0;
  Seq s = {0, 0, 0};
  Blocks k = {0, 0, 0};
  if (tid < entries) {
    int hi = p.batch - 1;
    while (b < hi) {
      const int mid = (b + hi + 1) >> 1;
      if (entry_s[mid] <= tid) b = mid;
      else hi = mid - 1;
    }
    s = Seq{row0_s[b], T_s[b], L_s[b]};
    e = tile = tid - entry_s[b];
    if (MASS) {
      tile = key_tile(key_tiles_of(p, s, a.kb_log2), e);
      const Tokens t = tokens_of(p, s, tile << a.kb_log2, 1 << a.kb_log2);
      k.window0 = t.first / a.block_tokens;
      n = ((t.last + a.block_tokens - 1) / a.block_tokens - k.window0) * a.head_chunks;
    } else {
      k = blocks_of(p, s, e, a.kb_log2);
      n = k.count();
      atomicMax(&most_s[b], n);
      atomicMax(&longest_s, n);
    }
  }
  const int before = scan(n), total = warp_sum[32];
  stage_s[tid] = before;
  if (tid == 0) stage_s[kPlanThreads] = total;
  __syncthreads();
  // ---- which way: warp w weighs chunks of at most longest / (w + 1) stages
  const int longest = longest_s;
  const long long stages = (long long)total * heads;
  int run = 0;
  if (!MASS) {
    float rows = 0.f;
    for (int w = 0; w < 32; w++) rows += seen_s[w];
    constexpr float kHbm = 6500.f;  // bytes per ns
    const float once = rows * (float)p.nkh * (float)p.hd * 4.f;  // bytes, K and V
    const int size = (longest + warp) / (warp + 1);
    int pieces = 0, cut = 0;
    for (int i = lane; i < p.batch; i += 32) {
      const int m = ((i + 1 < p.batch ? entry_s[i + 1] : entries) - entry_s[i]) * heads;
      const int parts = (most_s[i] + size - 1) / size;
      pieces += m * parts;
      if (parts > 1) cut += m * parts;
    }
    pieces = __reduce_add_sync(0xffffffffu, pieces);
    cut = __reduce_add_sync(0xffffffffu, cut);
    if (lane == 0) {
      const float waves = (float)((pieces + a.pairs - 1) / a.pairs);
      costs[warp] = cut > a.max_slots ? 3e38f : fmaxf(waves * (float)(size + kLead), once / kHbm / a.stage_ns) + (cut > 0 ? kJoinCost : 0);
    }
    __syncthreads();
    const float moved = (float)stages * a.stage_bytes;
    // (90 MB of the 126 MB L2, beside what else passes through it)
    const float floor_runs = (once > 90e6f ? fmaxf(moved, once) : once) / kHbm / a.stage_ns;
    float best = fmaxf(((float)stages + (float)kLead * (float)items) / (float)a.pairs + kLead, floor_runs) + kJoinCost;
    for (int w = 0; w < 32; w++)
      if (costs[w] < best) best = costs[w], run = (longest + w) / (w + 1);
  }
  if (run > 0) {
    // ---- chunks: pieces before each sequence, places of partial results
    int parts = 0;
    if (tid < p.batch) parts = (most_s[tid] + run - 1) / run;
    const int pieces0 = scan(tiles * heads * parts);
    const int pieces = warp_sum[32];
    __syncthreads();
    place_s[tid] = scan(parts > 1 ? tiles * heads * parts : 0);
    stage_s[tid] = pieces0;  // (the stages are not needed any more)
    for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(w, pieces, a.pairs, 0);
    __syncthreads();
    if (tid < entries) {
      const int of = (b + 1 < p.batch ? entry_s[b + 1] : entries) - entry_s[b];
      const int all = (most_s[b] + run - 1) / run, split = min(all, n);
      for (int head = 0; head < heads; head++) {
        const int kvh = head / a.halves, half = head - kvh * a.halves, slot = place_s[b] + (head * of + e) * all;
        for (int c = 0; c < all; c++) {
          Piece d;
          d.b = b, d.head = head, d.tile = tile, d.row0 = s.row0, d.T = s.T, d.L = s.L;
          d.j0 = c < split ? n * c / split : 0;
          d.j1 = c < split ? n * (c + 1) / split : 0;
          d.slot = split > 1 ? slot + c : -1;
          d.sinks = k.sinks, d.skip = k.window0 - k.sinks, d.pad = 0;
          a.pieces[stage_s[b] + (kvh * all + c) * of * a.halves + e * a.halves + half] = d;
        }
        if (split > 1) a.cuts[atomicAdd(&cut_count, 1)] = Cut{b, head, tile, s.row0, s.T, split, slot, slot + 1, 1};
      }
    }
  } else {
    // ---- runs
    const long long length = stages + (long long)kLead * items;
    const int pairs = (int)min((long long)a.pairs, length);
    if (tid < entries) {
      const int next = b + 1 < p.batch ? entry_s[b + 1] : entries, of = next - entry_s[b];
      const int first = stage_s[entry_s[b]], all = (next < entries ? stage_s[next] : total) - first;
      for (int head = 0; head < heads; head++) {
        const int i = entry_s[b] * heads + head * of + e;
        const long long at = (long long)first * heads + (long long)head * all + (before - first) + (long long)kLead * i;
        emit_runs<MASS>(a, s, b, head, tile, k, i, items, at, n, length, pairs, &cut_count);
      }
    }
  }
  __syncthreads();
  if (tid == 0) a.plan->cuts = cut_count;
}

// Any call: the same with the sequences and the tiles' counts in global memory.
template <bool MASS>
__global__ void __launch_bounds__(kPlanThreads) chunk_plan_kernel(const PlanParams a) {
  __shared__ long long warp_sum[32][4];
  __shared__ float costs[32];
  __shared__ int cut_count, run_s;
  const ChunkParams& p = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long cap = MASS ? min((long long)p.max_pages * p.page_size, p.mass_stride) : (long long)p.max_pages * p.page_size;
  const int heads = p.nkh * a.halves;
  // masses: the key tile of a sequence's entry, and its row blocks
  auto key_tile = [&](const Blocks& k, int e) { return e < k.sinks ? e : e + k.window0 - k.sinks; };
  auto row_blocks = [&](const Seq& s, int tile, int& first) {
    const Tokens t = tokens_of(p, s, tile << a.kb_log2, 1 << a.kb_log2);
    first = t.first / a.block_tokens;
    return ((t.last + a.block_tokens - 1) / a.block_tokens - first) * a.head_chunks;
  };
  pdl_wait_primary();
  pdl_launch_dependents();
  if (tid == 0) cut_count = 0;
  // ---- sequences: entries (tiles of one head) and items before each, the most stages of a tile
  long long entries_all = 0;
  int entries = 0, items = 0, longest = 0;
  float rows_seen = 0.f;  // rows of the cache that have to be read, over the sequences (for one kv head)
  for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    long long x[2] = {0, 0}, all[2];
    int most = 0;
    if (b < p.batch) {
      const Seq s = seq_of(p, b, cap);
      if (s.T > 0) {
        const int tiles = MASS ? key_tiles_of(p, s, a.kb_log2).count() : tiles_of(p, s);
        x[0] = tiles;
        x[1] = (long long)tiles * heads;
        if (!MASS) most = max(blocks_of(p, s, 0, a.kb_log2).count(), blocks_of(p, s, tiles - 1, a.kb_log2).count());
        rows_seen += (float)(s.L - first_in_window(p, s.base()));
      }
    }
    const int mine = (int)x[0], mine_items = (int)x[1];
    block_scan<2>(x, all, reinterpret_cast<long long(*)[2]>(warp_sum));
    if (b < p.batch) a.seqs[b] = make_int4(entries + (int)x[0] - mine, items + (int)x[1] - mine_items, most, 0);
    entries_all += all[0];
    entries += (int)all[0];
    items += (int)all[1];
    longest = max(longest, most);
  }
  if (tid == 0) a.seqs[p.batch] = make_int4(entries, items, 0, 0);
  {  // over the block
    __shared__ int most_s;
    __shared__ float seen_s;
    if (tid == 0) most_s = 0, seen_s = 0.f;
    __syncthreads();
    atomicMax(&most_s, longest);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) rows_seen += __shfl_xor_sync(0xffffffffu, rows_seen, o);
    if (lane == 0) costs[warp] = rows_seen;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < 32; w++) seen_s += costs[w];
    __syncthreads();
    longest = most_s;
    rows_seen = seen_s;
  }
  if (entries_all > a.max_entries) {  // (the same for all threads)
    if (tid == 0) a.plan->cuts = 0, atomicExch(p.err, G4A_DEVERR_TREE);
    for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
    for (int b = tid; MASS && b < p.batch; b += kPlanThreads) a.seqs[b] = make_int4(0, -1, 0, 0);
    return;
  }
  // ---- stages of all earlier entries
  long long total = 0;  // of one head
  for (int e0 = 0; e0 < entries; e0 += kPlanThreads) {
    const int e = e0 + tid;
    long long x[1] = {0}, all[1];
    if (e < entries) {
      const int b = find_seq(a.seqs, p.batch, e, false);
      const Seq s = seq_of(p, b, cap);
      int first;
      x[0] = MASS ? row_blocks(s, key_tile(key_tiles_of(p, s, a.kb_log2), e - a.seqs[b].x), first)
                  : blocks_of(p, s, e - a.seqs[b].x, a.kb_log2).count();
    }
    const long long mine = x[0];
    block_scan<1>(x, all, reinterpret_cast<long long(*)[1]>(warp_sum));
    if (e < entries) a.entries[e] = total + x[0] - mine;
    total += all[0];
  }
  __syncthreads();
  if (items == 0) {
    if (tid == 0) a.plan->cuts = 0;
    for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
    return;
  }
  // ---- which way: warp k weighs chunks of at most longest / (k + 1) stages
  const long long stages = total * heads;
  const float hbm = 6500.f;  // bytes per ns
  const float once = rows_seen * (float)p.nkh * (float)p.hd * 4.f;  // bytes, K and V
  const float floor_once = once / hbm / a.stage_ns;
  if (!MASS) {
    const int run = (longest + warp) / (warp + 1);
    long long pieces = 0, cut = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int n = a.seqs[b + 1].y - a.seqs[b].y;
      if (n == 0) continue;
      const int parts = (a.seqs[b].z + run - 1) / run;
      pieces += (long long)n * parts;
      if (parts > 1) cut += (long long)n * parts;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      pieces += __shfl_xor_sync(0xffffffffu, pieces, o);
      cut += __shfl_xor_sync(0xffffffffu, cut, o);
    }
    if (lane == 0) {
      const float waves = (float)((pieces + a.pairs - 1) / a.pairs);
      costs[warp] = cut > a.max_slots ? 3e38f : fmaxf(waves * (float)(run + kLead), floor_once) + (cut > 0 ? kJoinCost : 0);
    }
  }
  __syncthreads();
  if (tid == 0) {
    const float moved = (float)stages * a.stage_bytes;
    // (90 MB of the 126 MB L2, beside what else passes through it)
    const float floor_runs = (once > 90e6f ? fmaxf(moved, once) : once) / hbm / a.stage_ns;
    float best = fmaxf(((float)stages + (float)kLead * (float)items) / (float)a.pairs + kLead, floor_runs) + kJoinCost;
    int run = 0;
    for (int k = 0; k < (MASS ? 0 : 32); k++)
      if (costs[k] < best) best = costs[k], run = (longest + k) / (k + 1);
    run_s = run;
  }
  __syncthreads();
  const int run = run_s;
  if (run > 0) {
    // ---- chunks: pieces before each sequence, and places of partial results (kept at its first tile)
    int before = 0;
    long long slots = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
      const int b = b0 + tid;
      long long x[2] = {0, 0}, all[2];
      bool any = false;
      if (b < p.batch) {
        const int n = a.seqs[b + 1].y - a.seqs[b].y, parts = (a.seqs[b].z + run - 1) / run;
        any = n > 0;
        x[0] = (long long)n * parts;
        x[1] = parts > 1 ? x[0] : 0;
      }
      const long long mine = x[0], mine_slots = x[1];
      block_scan<2>(x, all, reinterpret_cast<long long(*)[2]>(warp_sum));
      if (any) {
        a.seqs[b].w = before + (int)(x[0] - mine);
        a.entries[a.seqs[b].x] = slots + x[1] - mine_slots;
      }
      before += (int)all[0];
      slots += all[1];
    }
    for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(w, before, a.pairs, 0);
    __syncthreads();
    for (int i = tid; i < items; i += kPlanThreads) {
      const int b = find_seq(a.seqs, p.batch, i, true);
      const int4 q = a.seqs[b];
      const Seq s = seq_of(p, b, cap);
      const int tiles = a.seqs[b + 1].x - q.x, local = i - q.y;
      const int head = local / tiles, tile = local - head * tiles, kvh = head / a.halves, half = head - kvh * a.halves;
      const Blocks k = blocks_of(p, s, tile, a.kb_log2);
      const int n = k.count(), all = (q.z + run - 1) / run, parts = min(all, n);
      const int slot = (int)a.entries[q.x] + local * all;
      for (int c = 0; c < all; c++) {
        Piece d;
        d.b = b, d.head = head, d.tile = tile, d.row0 = s.row0, d.T = s.T, d.L = s.L;
        d.j0 = c < parts ? (int)((long long)n * c / parts) : 0;
        d.j1 = c < parts ? (int)((long long)n * (c + 1) / parts) : 0;
        d.slot = parts > 1 ? slot + c : -1;
        d.sinks = k.sinks, d.skip = k.window0 - k.sinks, d.pad = 0;
        a.pieces[q.w + (kvh * all + c) * tiles * a.halves + tile * a.halves + half] = d;
      }
      if (parts > 1) a.cuts[atomicAdd(&cut_count, 1)] = Cut{b, head, tile, s.row0, s.T, parts, slot, slot + 1, 1};
    }
    __syncthreads();
    if (tid == 0) a.plan->cuts = cut_count;
    return;
  }
  // ---- runs
  const long long length = stages + (long long)kLead * items;
  const int pairs = (int)min((long long)a.pairs, length);
  for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
  __syncthreads();
  for (int i = tid; i < items; i += kPlanThreads) {
    const int b = find_seq(a.seqs, p.batch, i, true);
    const Seq s = seq_of(p, b, cap);
    const int e0 = a.seqs[b].x, tiles = a.seqs[b + 1].x - e0, local = i - a.seqs[b].y;
    const int head = local / tiles, e = local - head * tiles;
    const long long first = a.entries[e0], mine = (a.seqs[b + 1].x < entries ? a.entries[e0 + tiles] : total) - first;
    const long long at = first * heads + head * mine + (a.entries[e0 + e] - first) + (long long)kLead * i;
    int tile = e;
    Blocks k = {0, 0, 0};
    if (MASS) {
      tile = key_tile(key_tiles_of(p, s, a.kb_log2), e);
      row_blocks(s, tile, k.window0);
    } else {
      k = blocks_of(p, s, e, a.kb_log2);
    }
    const long long n = (e0 + e + 1 < entries ? a.entries[e0 + e + 1] : total) - a.entries[e0 + e];
    emit_runs<MASS>(a, s, b, head, tile, k, i, items, at, n, length, pairs, &cut_count);
  }
  __syncthreads();
  if (tid == 0) a.plan->cuts = cut_count;
}

}  // namespace

cudaError_t g4a_chunk_plan_launch(g4a_ctx* ctx, const PlanParams& a, bool masses, long long entries) {
  const bool small = a.c.batch <= kPlanThreads && entries <= kPlanThreads;
  return g4a_launch(small ? (masses ? chunk_plan_small_kernel<true> : chunk_plan_small_kernel<false>)
                          : (masses ? chunk_plan_kernel<true> : chunk_plan_kernel<false>),
                    dim3(1), dim3(kPlanThreads), 0, ctx->stream, true, a);
}
