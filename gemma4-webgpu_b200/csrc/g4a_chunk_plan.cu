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
// It takes 6 us, latency: the loads of the lengths, and then sums over the block that wait for one another.  With one
// thread for all pieces of a tile, and runs for all pairs whatever their parts cost to join, 8 tokens over 8,000 rows took
// 49 us, the whole call, instead of 23.
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

// An item of a list that is cut into equal runs: it has n stages, kLead in front of them, and begins at `at`.
struct Item {
  int i, b, head, tile;
  Seq s;
  Blocks k;
  long long at, n;
};
// Run w is [w length / pairs, (w + 1) length / pairs) of the list.  A piece of pair w of item i lies at i + w in the list
// of pieces, so a pair's lie together (with holes between the pairs).  A pair has at most one piece that goes on from the
// pair before (its result in place 2 w) and one that the next goes on with (2 w + 1).  A thread for each item writes its
// first piece, a thread for each pair the one that goes on: one thread for all pieces of an item took 0.4 us for each.
struct Runs {
  long long length;
  int pairs, items;
  __device__ __forceinline__ long long begin(int w) const { return quot((long long)w * length, pairs); }
  __device__ __forceinline__ int owner(long long x) const { return (int)quot((x + 1) * pairs - 1, length); }
};
__device__ __forceinline__ void put_piece(const PlanParams& a, const Runs& r, const Item& t, int w, long long j0, int last, bool first_of_pair) {
  Piece d;
  d.b = t.b, d.head = t.head, d.tile = t.tile, d.row0 = t.s.row0, d.T = t.s.T, d.L = t.s.L;
  d.j0 = (int)j0;
  d.j1 = w == last ? (int)t.n : (int)(r.begin(w + 1) - t.at - kLead);
  d.slot = j0 > 0 ? 2 * w : w == last ? -1 : 2 * w + 1;
  d.sinks = t.k.sinks, d.skip = t.k.window0 - t.k.sinks, d.pad = 0;
  a.pieces[t.i + w] = d;
  if (first_of_pair) a.plan->pair[w].x = t.i + w;
  // the pair's last piece: the item goes on in the next pair, or the next item begins there
  if (w < last || t.i + 1 == r.items || r.owner(t.at + t.n + 2 * kLead) > w) a.plan->pair[w].y = t.i + w + 1;
}
template <bool MASS>
__device__ __forceinline__ void put_first(const PlanParams& a, const Runs& r, const Item& t, int* cut_count) {
  const int w0 = r.owner(t.at + kLead), last = r.owner(t.at + kLead + t.n - 1);
  put_piece(a, r, t, w0, 0, last, t.i == 0 || r.owner(t.at - 1) < w0);
  if (MASS) a.parts[t.i] = make_int2(w0, last - w0 + 1);
  else if (last > w0)
    a.cuts[atomicAdd(cut_count, 1)] = Cut{t.b, t.head, t.tile, t.s.row0, t.s.T, last - w0 + 1, 2 * w0 + 1, 2 * (w0 + 1), 2};
}
// t: the item in which run w begins
__device__ __forceinline__ void put_next(const PlanParams& a, const Runs& r, const Item& t, int w) {
  const long long j0 = r.begin(w) - t.at - kLead;
  if (j0 > 0) put_piece(a, r, t, w, j0, r.owner(t.at + kLead + t.n - 1), true);
}
// What joining `parts` partial results costs, in stages.
__device__ __forceinline__ float join_cost(const PlanParams& a, float parts) {
  return parts == 0.f ? 0.f : (kJoinNs + parts * a.part_bytes / kJoinRate) / a.stage_ns;
}
// The last of [0, n) for which f is not above x (f rises, f(0) <= x).
template <typename F>
__device__ __forceinline__ int last_not_above(int n, long long x, F f) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (f(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A small call: up to kPlanThreads sequences and as many tiles, one to a thread, all in shared memory.
template <bool MASS>
__global__ void __launch_bounds__(kPlanThreads) chunk_plan_small_kernel(const PlanParams a) {
  __shared__ int warp_sum[33], row0_s[kPlanThreads], T_s[kPlanThreads], L_s[kPlanThreads], entry_s[kPlanThreads + 1];
  __shared__ int most_s[kPlanThreads], stage_s[kPlanThreads + 1], place_s[kPlanThreads];
  __shared__ float costs[32], seen_s[32], rows_s[32];
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
  float rows = (float)mine.T * (float)p.group;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    seen += __shfl_xor_sync(0xffffffffu, seen, o);
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
  }
  if (lane == 0) seen_s[warp] = seen, rows_s[warp] = rows;
  entry_s[tid] = scan(tiles);
  const int entries = warp_sum[32], items = entries * heads;
  if (tid == 0) entry_s[kPlanThreads] = entries;
  for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
  if (MASS && tid <= p.batch) a.seqs[tid] = make_int4(0, (tid < p.batch && tid < kPlanThreads ? entry_s[tid] : entries) * heads, 0, 0);
  __syncthreads();
  if (items == 0 || entries > a.max_entries) {
    if (tid == 0) a.plan->cuts = 0;
    if (items != 0) {  // (no items: the masses' rows fade all the same)
      if (tid == 0) atomicExch(p.err, G4A_DEVERR_TREE);
      if (MASS && tid < p.batch) a.seqs[tid] = make_int4(0, -1, 0, 0);
    }
    return;
  }
  // ---- tiles: a thread's sequence is the last one whose entries begin at or before it (those without any share a begin)
  int n = 0;
  if (tid < entries) {
    const int b = last_not_above(p.batch, tid, [&](int m) { return (long long)entry_s[m]; }), e = tid - entry_s[b];
    const Seq s = {row0_s[b], T_s[b], L_s[b]};
    if (MASS) {
      const Tokens t = tokens_of(p, s, key_tile(key_tiles_of(p, s, a.kb_log2), e) << a.kb_log2, 1 << a.kb_log2);
      n = ((t.last + a.block_tokens - 1) / a.block_tokens - t.first / a.block_tokens) * a.head_chunks;
    } else {
      n = blocks_of(p, s, e, a.kb_log2).count();
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
  int run = 0, used = a.pairs;
  if (!MASS) {
    float seen_all = seen_s[lane], rows_all = rows_s[lane];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      seen_all += __shfl_xor_sync(0xffffffffu, seen_all, o);
      rows_all += __shfl_xor_sync(0xffffffffu, rows_all, o);
    }
    const float full = fminf(1.f, rows_all / ((float)entries * kTileRows));  // rows that a tile has
    constexpr float kHbm = 6500.f;  // bytes per ns
    const float once = seen_all * (float)p.nkh * (float)p.hd * 4.f;  // bytes, K and V
    const float per_ns = 1.f / a.stage_ns, floor_once = once * (per_ns / kHbm);
    const int size = (longest + warp) / (warp + 1);
    int pieces = 0, cut = 0;
#pragma unroll 1
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
      costs[warp] = cut > a.max_slots ? 3e38f : fmaxf(waves * (float)(size + kLead), floor_once) + join_cost(a, (float)cut * full);
    }
    __syncthreads();
    // the cheapest chunks
    const uint32_t mine = __float_as_uint(costs[lane]);  // (not negative: ordered as whole numbers)
    const uint32_t least = __reduce_min_sync(0xffffffffu, mine);
    const int k = __ffs(__ballot_sync(0xffffffffu, mine == least)) - 1;
    // runs: fewer, longer ones where the parts would cost more than the keys (length / pairs + pairs x a part's cost is
    // least where both are the same)
    const float length = (float)stages + (float)kLead * (float)items;
    used = max(1, min(a.pairs, (int)sqrtf(length * a.stage_ns * kJoinRate / (2.f * a.part_bytes * full))));
    // (90 MB of the 126 MB L2, beside what else passes through it)
    const float floor_runs = once > 90e6f ? fmaxf((float)stages * a.stage_bytes * (per_ns / kHbm), floor_once) : floor_once;
    const float runs = fmaxf(length / (float)used + kLead, floor_runs) + join_cost(a, (float)(used + min(items, used)) * full);
    if (__uint_as_float(least) < runs) run = (longest + k) / (k + 1);
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
    __syncthreads();
    for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(w, pieces, a.pairs, 0);
    const int most = (longest + run - 1) / run;
    for (int x = tid; x < entries * heads * most; x += kPlanThreads) {  // (entry, head, chunk)
      const int y = x / most, c = x - y * most, at_e = y / heads, head = y - at_e * heads;
      const int m = last_not_above(p.batch, at_e, [&](int i) { return (long long)entry_s[i]; });
      const int of = (m + 1 < p.batch ? entry_s[m + 1] : entries) - entry_s[m], t = at_e - entry_s[m];
      const int all = (most_s[m] + run - 1) / run;
      if (c >= all) continue;
      const Seq q = {row0_s[m], T_s[m], L_s[m]};
      const Blocks blocks = blocks_of(p, q, t, a.kb_log2);
      const int count = blocks.count(), split = min(all, count);
      const int kvh = head / a.halves, half = head - kvh * a.halves, slot = place_s[m] + (head * of + t) * all;
      Piece d;
      d.b = m, d.head = head, d.tile = t, d.row0 = q.row0, d.T = q.T, d.L = q.L;
      d.j0 = c < split ? count * c / split : 0;
      d.j1 = c < split ? count * (c + 1) / split : 0;
      d.slot = split > 1 ? slot + c : -1;
      d.sinks = blocks.sinks, d.skip = blocks.window0 - blocks.sinks, d.pad = 0;
      a.pieces[stage_s[m] + (kvh * all + c) * of * a.halves + t * a.halves + half] = d;
      if (c == 0 && split > 1) a.cuts[atomicAdd(&cut_count, 1)] = Cut{m, head, t, q.row0, q.T, split, slot, slot + 1, 1};
    }
  } else {
    // ---- runs
    Runs r;
    r.length = stages + (long long)kLead * items, r.items = items, r.pairs = (int)min((long long)used, r.length);
    // tile e of head `head` of sequence b
    auto item_of = [&](int b, int head, int e) {
      Item t;
      const int next = b + 1 < p.batch ? entry_s[b + 1] : entries, of = next - entry_s[b], at_e = entry_s[b] + e;
      const int first = stage_s[entry_s[b]], all = (next < entries ? stage_s[next] : total) - first;
      t.i = entry_s[b] * heads + head * of + e, t.b = b, t.head = head;
      t.s = Seq{row0_s[b], T_s[b], L_s[b]};
      t.n = (at_e + 1 < entries ? stage_s[at_e + 1] : total) - stage_s[at_e];
      t.at = (long long)first * heads + (long long)head * all + (stage_s[at_e] - first) + (long long)kLead * t.i;
      t.k = Blocks{0, 0, 0};
      t.tile = e;
      if (MASS) {
        t.tile = key_tile(key_tiles_of(p, t.s, a.kb_log2), e);
        t.k.window0 = tokens_of(p, t.s, t.tile << a.kb_log2, 1 << a.kb_log2).first / a.block_tokens;
      } else {
        t.k = blocks_of(p, t.s, e, a.kb_log2);
      }
      return t;
    };
    for (int x = tid; x < items; x += kPlanThreads) {  // (entry, head)
      const int at_e = x / heads, head = x - at_e * heads;
      const int of_b = last_not_above(p.batch, at_e, [&](int m) { return (long long)entry_s[m]; });
      put_first<MASS>(a, r, item_of(of_b, head, at_e - entry_s[of_b]), &cut_count);
    }
    for (int w = tid + 1; w < r.pairs; w += kPlanThreads) {
      const long long x = r.begin(w);
      auto seq_at = [&](int m) {
        return entry_s[m] < entries ? (long long)stage_s[entry_s[m]] * heads + (long long)kLead * heads * entry_s[m] : r.length;
      };
      const int of_b = last_not_above(p.batch, x, seq_at);
      const int next = of_b + 1 < p.batch ? entry_s[of_b + 1] : entries, of = next - entry_s[of_b], first = stage_s[entry_s[of_b]];
      const long long per = (next < entries ? stage_s[next] : total) - first + (long long)kLead * of, in = x - seq_at(of_b);
      const int head = (int)quot(in, per);
      const long long rest = in - head * per;
      const int e = last_not_above(of, rest, [&](int m) { return (long long)(stage_s[entry_s[of_b] + m] - first) + (long long)kLead * m; });
      put_next(a, r, item_of(of_b, head, e), w);
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
      costs[warp] = cut > a.max_slots ? 3e38f : fmaxf(waves * (float)(run + kLead), floor_once) + join_cost(a, (float)cut);
    }
  }
  __syncthreads();
  if (tid == 0) {
    const float moved = (float)stages * a.stage_bytes;
    // (90 MB of the 126 MB L2, beside what else passes through it)
    const float floor_runs = (once > 90e6f ? fmaxf(moved, once) : once) / hbm / a.stage_ns;
    float best = fmaxf(((float)stages + (float)kLead * (float)items) / (float)a.pairs + kLead, floor_runs) + join_cost(a, 2.f * (float)a.pairs);
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
  Runs r;
  r.length = stages + (long long)kLead * items, r.items = items, r.pairs = (int)min((long long)a.pairs, r.length);
  for (int w = tid; w < a.pairs; w += kPlanThreads) a.plan->pair[w] = make_int4(0, 0, 1, 0);
  __syncthreads();
  auto item_of = [&](int b, int head, int e) {
    Item t;
    const int e0 = a.seqs[b].x, next = a.seqs[b + 1].x, of = next - e0;
    const long long first = a.entries[e0], all = (next < entries ? a.entries[next] : total) - first;
    t.i = a.seqs[b].y + head * of + e, t.b = b, t.head = head;
    t.s = seq_of(p, b, cap);
    t.n = (e0 + e + 1 < entries ? a.entries[e0 + e + 1] : total) - a.entries[e0 + e];
    t.at = first * heads + head * all + (a.entries[e0 + e] - first) + (long long)kLead * t.i;
    t.k = Blocks{0, 0, 0};
    t.tile = e;
    if (MASS) {
      t.tile = key_tile(key_tiles_of(p, t.s, a.kb_log2), e);
      (void)row_blocks(t.s, t.tile, t.k.window0);
    } else {
      t.k = blocks_of(p, t.s, e, a.kb_log2);
    }
    return t;
  };
  for (int i = tid; i < items; i += kPlanThreads) {
    const int b = find_seq(a.seqs, p.batch, i, true), of = a.seqs[b + 1].x - a.seqs[b].x, local = i - a.seqs[b].y;
    put_first<MASS>(a, r, item_of(b, local / of, local % of), &cut_count);
  }
  for (int w = tid + 1; w < r.pairs; w += kPlanThreads) {
    const long long x = r.begin(w);
    auto seq_at = [&](int m) {
      return a.seqs[m].x < entries ? a.entries[a.seqs[m].x] * heads + (long long)kLead * a.seqs[m].y : r.length;
    };
    const int b = last_not_above(p.batch, x, seq_at), e0 = a.seqs[b].x, next = a.seqs[b + 1].x;
    const long long first = a.entries[e0], per = (next < entries ? a.entries[next] : total) - first + (long long)kLead * (next - e0);
    const long long in = x - seq_at(b), head = quot(in, per), rest = in - head * per;
    const int e = last_not_above(next - e0, rest, [&](int m) { return a.entries[e0 + m] - first + (long long)kLead * m; });
    put_next(a, r, item_of(b, (int)head, e), w);
  }
  __syncthreads();
  if (tid == 0) a.plan->cuts = cut_count;
}

}  // namespace

cudaError_t g4a_chunk_plan_launch(g4a_ctx* ctx, const PlanParams& a, bool masses, long long entries) {
  // (the small kernel adds up a head's stages in 32 bits)
  const ChunkParams& p = a.c;
  const long long rows = (long long)p.page_size * p.max_pages;
  const long long most = masses ? ((long long)p.tokens / a.block_tokens + 2) * a.head_chunks : (rows >> a.kb_log2) + 3;
  const bool small = p.batch <= kPlanThreads && entries <= kPlanThreads && entries * most <= 0x7fffffffll;
  return g4a_launch(small ? (masses ? chunk_plan_small_kernel<true> : chunk_plan_small_kernel<false>)
                          : (masses ? chunk_plan_kernel<true> : chunk_plan_kernel<false>),
                    dim3(1), dim3(kPlanThreads), 0, ctx->stream, true, a);
}
