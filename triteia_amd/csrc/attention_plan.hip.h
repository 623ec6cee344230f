// The work list of paged attention over a batch, made once for a forward pass and read by every layer of it.
//
// Sequence b brings tokens q_starts[b] .. q_starts[b + 1] - 1 and has kv_lens[b] tokens in the cache, the new ones last.  For a head of the
// cache its rows are (token, head of the group) pairs, token major.  Sequences of few rows go to the list of row tiles (one
// wavefront's MFMA columns), the others to the list of 128-row tiles.  A tile whose part of the cache is long is cut into shares of whole
// 64-token blocks, so that every list has work for the whole chip; a share's result goes to scratch and a tile's shares are joined by a launch behind.
// Lengths stay on the device: what the host knows are upper bounds, from which it sizes the lists and the grids.
//
// One workgroup of two wavefronts, a list each, so that nothing but the sequences' lengths in LDS is waited for: sums over the lanes, a lane finds the
// sequence of a tile by a binary search.  Tokens behind the last sequence get tiles without keys, whose rows are zeros.  Every number read from the
// device is clamped and offsets that do not ascend are made to, so that every row has one tile and no list passes its end.
// Bound by latency: 6.4 us for one sequence, 8.2 for a step's 26 of which two are long (14.2 with 1024 threads on one list after the other, whose barriers
// and shuffles were the time), 10.9 for 64, 15.7 for four prompts of 500 tokens and 64 heads over 8 (108 tiles), all of which are also put in order.
#pragma once
#include "lora_routed.hip.h"

namespace triteia_hip {

constexpr int kAttnBlock = 64;         // tokens of a block: shares begin and end on its multiples
constexpr int kAttnTileRows = 128;     // rows of a tile of the long list
constexpr int kAttnWaves = 8;          // at most, of a workgroup with few rows
constexpr int kAttnSorted = 256;       // lists of up to this many tiles begin with the longest
constexpr int kAttnMaxSeqs = 4096;
constexpr int kAttnMaxTokens = 0x7fffff80;   // a longer context is taken as this long, so that the end of its last block is still an int
constexpr int kAttnPlanThreads = 128;

// One share of one tile.
struct AttnItem {
  int seq, q_start, n_tokens, kv_len, tile, kv_begin, kv_end, part;   // part: of the scratch, -1: the whole tile
};
// A tile of several shares.
struct AttnJoin {
  int q_start, n_tokens, tile, first, n_parts, unused[3];
};

struct AttnList {
  int rows;              // rows of a tile
  int max_items, max_joins;
  long items, joins;     // where they start in the plan, in ints
  int slots, min_blocks; // workgroups that run side by side, and the least length of a share
  int waves;             // of a workgroup
  int rounds;            // lists of this many rounds of workgroups and more are not cut
  int max_parts;
};

struct AttnLayout {
  int n_seqs, n_tokens, group, kv_heads, causal, window;
  int short_rows;        // sequences of more rows go to the long list; 0x7fffffff: there is none
  AttnList list[2];      // short, long
  long ints;
};

// Everything that the host knows of a plan.
inline AttnLayout attn_layout(int n_seqs, int n_tokens, int heads, int kv_heads, int max_q, int causal, int window) {
  AttnLayout a = {};
  a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.group = heads / kv_heads, a.kv_heads = kv_heads, a.causal = causal, a.window = window;
  const long rows = (long)n_tokens * a.group, most = (long)(max_q < n_tokens ? max_q : n_tokens) * a.group;
  const long live = n_seqs + 1 < n_tokens ? n_seqs + 1 : n_tokens;      // sequences with tokens, and the tokens behind them
  const bool only_short = most <= 32;
  AttnList &s = a.list[0], &l = a.list[1];
  s.rows = only_short && most > 16 ? 32 : 16;
  a.short_rows = only_short ? 0x7fffffff : a.group <= 16 ? 16 : 0;       // (one token's heads fill more than a tile of 16: a long sequence)
  // A share is worth its scratch and its place in the joining launch from 1024 tokens on (short rows) or 512 (tiles: 26 sequences, two of 203 new
  // tokens on up to 2000, in e4m3, 59.5 / 49.2 / 62.7 us with 256 / 512 / 768; 3 of 100 on 3000 58.1 / 58.3 / 63.3, 8 of 300 on 300 36.1 / 21.4 / 21.5).
  s.min_blocks = 16, s.rounds = 4, l.slots = 512, l.min_blocks = 8, l.rounds = 2;
  l.rows = kAttnTileRows;
  const long tiles[2] = {only_short ? live + rows / s.rows : a.short_rows ? live : 0, only_short ? 0 : live + rows / l.rows};
  // Up to 128 workgroups with short rows: eight wavefronts, one a CU, so that a context is walked fast.  More: four, two a CU, one beginning or
  // ending while the other streams.  (us, eight / four: 32 of 500 tokens 8.0 / 8.7, 24 of 100000 cut into 256 / 512 215 / 220, 192 of up to 2000 in
  // e4m3 22.9 / 21.0, 2048 of up to 1000 112 / 100 and 81 / 58, 1280 of 34 21.5 / 13.2, 2048 of up to 4096 395 / 390.)
  s.waves = !only_short || tiles[0] * kv_heads > 128 ? 4 : kAttnWaves;
  s.slots = only_short && s.waves == 4 ? 512 : 256, l.waves = 4;
  for (int which = 0; which < 2; which++) {
    AttnList& x = a.list[which];
    // (as the kernel cuts them: into the shares of whole rounds of workgroups; a cut tile has two at least)
    const long units = tiles[which] * kv_heads, whole = units < (long)x.rounds * x.slots ? units : (long)x.rounds * x.slots;
    const long shares = (whole + x.slots - 1) / x.slots * x.slots / kv_heads;
    x.max_joins = (int)(tiles[which] < shares / 2 ? tiles[which] : shares / 2);
    x.max_parts = (int)(tiles[which] > 0 ? shares : 0);
    x.max_items = (int)(tiles[which] > shares ? tiles[which] : shares);
  }
  long at = 8;
  for (AttnList& x : a.list) {
    x.items = at, at += 8L * x.max_items;
    x.joins = at, at += 8L * x.max_joins;
  }
  a.ints = at;
  return a;
}

// Exclusive sums over a wavefront's lanes, and the total.
__device__ __forceinline__ int attn_scan(int v, int* total) {
  const int x = lane_sums(v);
  *total = __builtin_amdgcn_readlane(x, 63);
  return x - v;
}

struct AttnSeq {
  int start, n, kv;
};
// the tokens of the cache that some row of a tile sees, its beginning on a whole block
__device__ __forceinline__ void attn_range(const AttnSeq& s, int tile, int rows, const AttnLayout& a, int* lo, int* hi) {
  const uint32_t row = (uint32_t)tile * rows;            // (tokens times heads of a group are below 2^31)
  const int t0 = (int)(row / (uint32_t)a.group), t1 = min(s.n - 1, (int)((row + rows - 1) / (uint32_t)a.group));
  const long before = (long)s.kv - s.n;
  *hi = a.causal ? (int)max(0L, before + t1 + 1) : s.kv;
  *lo = a.window > 0 ? (int)max(0L, before + t0 - a.window + 1) / kAttnBlock * kAttnBlock : 0;
  *lo = min(*lo, *hi / kAttnBlock * kAttnBlock);
}

// grid 1, block kAttnPlanThreads
__global__ __launch_bounds__(kAttnPlanThreads) void attention_plan_kernel(const int* q_starts, const int* kv_lens, AttnLayout a, int* plan) {
  __shared__ int start[kAttnMaxSeqs + 1], count[kAttnMaxSeqs + 1], context[kAttnMaxSeqs + 1];
  __shared__ int tiles_ahead[2][kAttnMaxSeqs + 1];       // of each sequence, in each list
  __shared__ int order[2][kAttnSorted];
  __shared__ int crossed[kAttnPlanThreads / 64];
  bool back = false;                                     // an offset below the one ahead of it
  for (int b = threadIdx.x; b <= a.n_seqs; b += kAttnPlanThreads) {
    const bool rest = b == a.n_seqs;
    const int lo = b == 0 ? 0 : max(0, min(q_starts[b], a.n_tokens)), hi = rest ? a.n_tokens : max(0, min(q_starts[b + 1], a.n_tokens));
    back |= hi < lo;
    start[b] = lo, count[b] = hi - lo, context[b] = rest ? 0 : min(max(kv_lens[b], 0), kAttnMaxTokens);
  }
  const bool any_back = __any(back);
  if ((threadIdx.x & 63) == 0) crossed[threadIdx.x >> 6] = any_back;
  __syncthreads();
  bool mend = false;
#pragma unroll
  for (int w = 0; w < kAttnPlanThreads / 64; w++) mend |= crossed[w] != 0;
  if (mend) {                                            // offsets in no order: each as the largest up to it, so that every token has one place
    if (threadIdx.x == 0) {
      for (int b = 1; b <= a.n_seqs; b++) {
        start[b] = max(start[b], start[b - 1]);
        count[b - 1] = start[b] - start[b - 1];
      }
      count[a.n_seqs] = a.n_tokens - start[a.n_seqs];
    }
    __syncthreads();
  }
  const int which = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const AttnList& l = a.list[which];
  if (l.max_items == 0) {
    if (lane < 2) plan[2 * which + lane] = 0;
    return;
  }
  int* ahead = tiles_ahead[which];
  int tiles = 0;
  for (int b0 = 0; b0 <= a.n_seqs; b0 += 64) {
    const int b = b0 + lane;
    int mine = 0;
    if (b <= a.n_seqs) {
      const long rows = (long)count[b] * a.group;
      if (rows > 0 && (rows <= a.short_rows) == (which == 0)) mine = (int)((rows + l.rows - 1) / l.rows);
    }
    int all;
    const int before = attn_scan(mine, &all);
    if (b <= a.n_seqs) ahead[b] = tiles + before;
    tiles += all;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");        // (the wavefront's own list: its lanes run together)
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  struct Tile {
    int seq, tile, lo, hi, blocks;
    AttnSeq s;
  };
  auto at = [&](int i) {
    int lo = 0, hi = a.n_seqs;                                   // the last sequence that starts at or ahead of tile i
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (ahead[mid] <= i) lo = mid; else hi = mid - 1;
    }
    Tile t;
    t.seq = lo, t.tile = i - ahead[lo], t.s = {start[lo], count[lo], context[lo]};
    attn_range(t.s, t.tile, l.rows, a, &t.lo, &t.hi);
    t.blocks = (t.hi - t.lo + kAttnBlock - 1) / kAttnBlock;
    return t;
  };
  int mine[kAttnSorted / 64];                                    // blocks of tiles `lane`, 64 + lane, ..
#pragma unroll
  for (int k = 0; k < kAttnSorted / 64; k++) mine[k] = 64 * k + lane < tiles ? at(64 * k + lane).blocks : -1;
  // Few tiles: the least share with which all shares still run in as many rounds as the tiles would.
  int share = 0x7fffffff;
  const long units = (long)tiles * a.kv_heads;
  if (units < (long)l.rounds * l.slots) {
    const int most = (int)((units + l.slots - 1) / l.slots * l.slots / a.kv_heads);        // shares of one head
    auto sum_of = [&](auto f) {                                  // f of every tile's blocks
      long sum = 0;
#pragma unroll
      for (int k = 0; k < kAttnSorted / 64; k++) sum += mine[k] < 0 ? 0 : f(mine[k]);
      for (int i0 = kAttnSorted; i0 < tiles; i0 += 64) sum += i0 + lane < tiles ? f(at(i0 + lane).blocks) : 0;
      int total;
      attn_scan((int)min(sum, 0x7fffffffL / 64), &total);
      return total;
    };
    const int total = sum_of([](int blocks) { return blocks; });
    share = max(l.min_blocks, (total + most - 1) / max(most, 1));
    while (share <= total && sum_of([&](int blocks) { return max(1, (blocks + share - 1) / share); }) > most) share += (share + 7) / 8;
  }
  // longest first, so that the last workgroups to run are short ones
  if (tiles <= kAttnSorted) {
    int place[kAttnSorted / 64] = {};
#pragma unroll
    for (int k = 0; k < kAttnSorted / 64; k++) {
      for (int i = 64 * k; i < min(tiles, 64 * k + 64); i++) {
        const int other = __builtin_amdgcn_readlane(mine[k], i & 63);
#pragma unroll
        for (int n = 0; n < kAttnSorted / 64; n++) place[n] += other > mine[n] || (other == mine[n] && i < 64 * n + lane);
      }
    }
#pragma unroll
    for (int k = 0; k < kAttnSorted / 64; k++)
      if (64 * k + lane < tiles) order[which][place[k]] = 64 * k + lane;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }
  int n_items = 0, n_joins = 0, n_parts = 0;
  int end_items = l.max_items, end_joins = l.max_joins;          // (all have a place: the cut leaves no more shares than the host has counted)
  for (int i0 = 0; i0 < tiles; i0 += 64) {
    // (of long lists a sequence's last tile, its longest, first)
    const int i = i0 + lane >= tiles ? -1 : tiles <= kAttnSorted ? order[which][i0 + lane] : tiles - 1 - (i0 + lane);
    int splits = 0, per = 0;
    Tile t = {};
    if (i >= 0) {
      t = at(i);
      splits = max(1, (int)(((long)t.blocks + share - 1) / share));
      per = (t.blocks + splits - 1) / splits;
      splits = per > 0 ? max(1, (t.blocks + per - 1) / per) : 1;
    }
    int all_items, all_joins, all_parts;
    const int item = n_items + attn_scan(splits, &all_items);
    const int join = n_joins + attn_scan(splits > 1, &all_joins);
    const int part = n_parts + attn_scan(splits > 1 ? splits : 0, &all_parts);
    if (i >= 0 && (item + splits > l.max_items || (splits > 1 && join >= l.max_joins))) {
      end_items = min(end_items, item), end_joins = min(end_joins, join);
    } else if (i >= 0) {
      AttnItem* out = reinterpret_cast<AttnItem*>(plan + l.items) + item;
      for (int p = 0; p < splits; p++)
        out[p] = AttnItem{t.seq, t.s.start, t.s.n, t.s.kv, t.tile, t.lo + p * per * kAttnBlock, splits == 1 ? t.hi : min(t.hi, t.lo + (p + 1) * per * kAttnBlock),
                          splits == 1 ? -1 : part + p};
      if (splits > 1) reinterpret_cast<AttnJoin*>(plan + l.joins)[join] = AttnJoin{t.s.start, t.s.n, t.tile, part, splits, {0, 0, 0}};
    }
    n_items += all_items, n_joins += all_joins, n_parts += all_parts;
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) end_items = min(end_items, __shfl_xor(end_items, d)), end_joins = min(end_joins, __shfl_xor(end_joins, d));
  if (lane == 0) plan[2 * which] = min(n_items, end_items), plan[2 * which + 1] = min(n_joins, end_joins);
}

}  // namespace triteia_hip
