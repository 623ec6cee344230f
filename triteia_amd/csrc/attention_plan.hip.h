// The work list of paged attention over a batch, made once for a forward pass and read by every layer of it.
//
// Sequence b brings tokens q_starts[b] .. q_starts[b + 1] - 1 and has kv_lens[b] tokens in the cache, the new ones last.  For a head of the
// cache its rows are (token, head of the group) pairs, token major.  Sequences of few rows go to the list of row tiles (one
// wavefront's MFMA columns), the others to the list of 128-row tiles.  A tile whose part of the cache is long is cut into shares of whole
// 64-token blocks, so that every list has work for the whole chip; a share's result goes to scratch and a tile's shares are joined by a launch behind.
// Lengths stay on the device: what the host knows are upper bounds, from which it sizes the lists and the grids.
//
// One workgroup of two wavefronts (with groups three), a list each, so that nothing but the sequences' lengths in LDS is waited for: sums over the lanes, a lane finds the
// sequence of a tile by a binary search.  Tokens behind the last sequence get tiles without keys, whose rows are zeros.  Every number read from the
// device is clamped and offsets that do not ascend are made to, so that every row has one tile and no list passes its end.
//
// Sequences in groups that share their first tokens (SHARED): group g is sequences group_starts[g] .. group_starts[g + 1] - 1, whose tables begin with the
// same pages.  Its sequences of up to 64 rows share, and those of up to 256 as long as a batch has few of them: of prefix_lens[g] tokens, those that all of their rows see, in whole
// blocks, are attended to once, by one more sequence, whose rows are all of their new tokens and whose context is the prefix, without a mask.  They themselves begin behind it, and each of
// their tiles is joined from its own shares and the shares of the prefix's tiles that hold its rows.  Prompts of the group walk their whole context: their tiles have the matrix cores busy
// either way, and in the prefix each of their rows is written in 32 bits and joined.  (us with them in the prefix or, where that does not pay, nothing shared, and without them: 64 requests of one token
// and one of 1000 behind 8192, 64 heads over 8, 539 and 424, three of 100 263 and 168; 48 and one of 3000 behind 2000, 32 + 32 heads, 366 and 260.  But one of 200 rows, 20 requests beside it, 51 and 61.)
// Where prompts stand between the others the prefix's rows are not adjacent, and the plan has a list of their tokens (`map`).
// Bound by latency: 6.4 us for one sequence, 8.2 for a step's 26 of which two are long (14.2 with 1024 threads on one list after the other, whose barriers
// and shuffles were the time), 10.9 for 64, 15.7 for four prompts of 500 tokens and 64 heads over 8 (108 tiles), all of which are also put in order.  With groups: five
// sequences of one 9.2, 64 13.3, 96 of six 18.9.
#pragma once
#include "lora_routed.hip.h"

namespace triteia_hip {

constexpr int kAttnBlock = 64;         // tokens of a block: shares begin and end on its multiples
constexpr int kAttnTileRows = 128;     // rows of a tile of the long list
constexpr int kAttnWaves = 8;          // at most, of a workgroup with few rows
constexpr int kAttnSorted = 256;       // lists of up to this many tiles begin with the longest
constexpr int kAttnMaxSeqs = 4096;
constexpr int kAttnMaxGroups = 1024;
constexpr int kAttnSolo = 512;         // groups' sequences times heads of the cache above which each gets a wavefront
constexpr int kAttnSharedRows = kAttnTileRows / 2;      // sequences of up to so many rows share a prefix,
// and of up to so many, if those of more than kAttnSharedRows have so many together.  (us, in the prefix and not: 64 of 80 rows beside 64 of 8 behind 4096, 64 heads over 8, 178 and 217, 32 of 160 beside
// 96 of 8 189 and 250; but 100 of 80 beside 100 of 4 behind 1500, 32 heads over 8, 175 and 146, and their scratch grows.)
constexpr int kAttnMostRows = 2 * kAttnTileRows, kAttnMoreRows = 6144;
constexpr int kAttnPrefixRows = 32;    // prefixes of up to so many rows are walked by all wavefronts of a workgroup
constexpr int kAttnRowBlocks = 16;     // blocks of a share of few rows, at least
constexpr int kAttnTileBlocks = 8;     // a share of a tile of 128 rows, at least
// Rounds of workgroups that groups' prompts are cut into, at most, if that leaves fewer slots idle (42 tiles of 96 blocks over 8 heads, 336 workgroups on 512 slots, as 126 of 32 206 -> 180 us;
// two groups of 3 prompts of 100 behind 12000, 64 heads over 8, 325 -> 274; three and four rounds give no more), and what a share costs ahead of its first block and in the join, in blocks.
constexpr int kAttnRounds = 2, kAttnShareBlocks = 4;
constexpr int kAttnHalf = 30;          // blocks of a workgroup, on half of the slots, up to which a prefix is not given all of them
constexpr int kAttnOwnBlocks = 8;      // so are few rows' own parts of more than so many blocks, in batches with groups
constexpr int kAttnMaxTokens = 0x7fffff80;   // a longer context is taken as this long, so that the end of its last block is still an int
constexpr int kAttnPlanThreads = 128;          // a wavefront for each list; of groups 192
constexpr int kAttnLists = 3;          // few rows, tiles of 128 rows, and long walks of few rows (groups only)

// One share of one tile.
struct AttnItem {
  int seq, q_start, n_tokens, kv_len, tile, kv_begin, kv_end, part;   // q_start: the first token, below zero of a list of them (attn_token); part: of the scratch, -1: the whole tile
};
// A tile of several shares, or of a group: the list of the group's prefix (-1: none), the prefix's first tile there and its row of the tile's sequence's first.
struct AttnJoin {
  int q_start, n_tokens, tile, first, n_parts, prefix_list, prefix_tile, prefix_row;
};

struct AttnList {
  int rows;              // rows of a tile
  int max_items, max_joins;
  long items, joins;     // where they start in the plan, in ints
  int slots, min_blocks; // workgroups that run side by side, and the least length of a share
  int waves;             // of a workgroup
  int rounds;            // lists of this many rounds of workgroups and more are not cut
  int max_parts;
  long prefixes;         // of each tile, its first share and their number (groups only)
};

struct AttnLayout {
  int n_seqs, n_tokens, group, kv_heads, causal, window, n_groups;
  int solo;              // short tiles: a wavefront each (groups only)
  int short_rows;        // sequences of more rows go to the long list; 0x7fffffff: there is none
  AttnList list[kAttnLists];      // short, long, walks
  int shared_rows;       // of prefixes, at most
  long map;              // tokens of prefixes whose rows are not adjacent (groups only)
  long ints;
};

// Everything that the host knows of a plan.
inline AttnLayout attn_layout(int n_seqs, int n_tokens, int heads, int kv_heads, int max_q, int causal, int window, int n_groups = 0) {
  AttnLayout a = {};
  a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.group = heads / kv_heads, a.kv_heads = kv_heads, a.causal = causal, a.window = window, a.n_groups = n_groups;
  const long rows = (long)n_tokens * a.group, most = (long)(max_q < n_tokens ? max_q : n_tokens) * a.group;
  const long live = n_seqs + 1 < n_tokens ? n_seqs + 1 : n_tokens;      // sequences with tokens, and the tokens behind them
  // (a group that shares has two sequences with tokens at least; its prefix has the rows of all of them)
  const long pairs = (n_seqs < n_tokens ? n_seqs : n_tokens) / 2, sharing = n_groups < pairs ? n_groups : pairs;
  a.shared_rows = (int)std::min(rows, (long)n_seqs * kAttnSharedRows + kAttnMoreRows);
  a.solo = sharing > 0 && a.group <= 16 && live * kv_heads > kAttnSolo;
  const bool only_short = most <= 32 && sharing == 0;
  AttnList &s = a.list[0], &l = a.list[1], &p = a.list[2];
  s.rows = only_short && most > 16 ? 32 : 16;
  a.short_rows = only_short ? 0x7fffffff : a.group <= 16 ? 16 : 0;       // (one token's heads fill more than a tile of 16: a long sequence)
  // A share is worth its scratch and its place in the joining launch from 1024 tokens on (short rows) or 512 (tiles: 26 sequences, two of 203 new
  // tokens on up to 2000, in e4m3, 59.5 / 49.2 / 62.7 us with 256 / 512 / 768; 3 of 100 on 3000 58.1 / 58.3 / 63.3, 8 of 300 on 300 36.1 / 21.4 / 21.5).
  s.min_blocks = kAttnRowBlocks, s.rounds = 4, l.slots = 512, l.min_blocks = kAttnTileBlocks, l.rounds = 2;
  l.rows = kAttnTileRows;
  p.rows = kAttnPrefixRows, p.slots = 512, p.min_blocks = kv_heads <= 8 ? 2 : 4, p.rounds = 2, p.waves = 4;
  long tiles[kAttnLists] = {only_short ? live + rows / s.rows : a.short_rows ? live : 0, only_short ? 0 : live + rows / l.rows, 0};
  long joined = 0, kept = 0;            // tiles of the long list that share a prefix, those and the prefixes'
  if (sharing > 0) {
    // (sequences and prefixes of the long list: of more rows than the others take.  A short prefix whose tokens are listed has a prompt in its group, and with it more rows than that.)
    joined = std::min(live, (long)a.shared_rows / (a.short_rows + 1)) + a.shared_rows / l.rows;
    const long prefixes = std::min(sharing, rows / (kAttnPrefixRows + 1)) + a.shared_rows / l.rows;
    kept = joined + prefixes;
    tiles[1] = std::min(live, rows / (a.short_rows + 1)) + rows / l.rows + prefixes;
    tiles[2] = sharing + live;
    l.min_blocks = 2;                  // (kAttnTileBlocks, and kAttnRowBlocks for walks, where it does not pay to share)
  }
  // Up to 128 workgroups with short rows: eight wavefronts, one a CU, so that a context is walked fast.  More: four, two a CU, one beginning or
  // ending while the other streams.  (us, eight / four: 32 of 500 tokens 8.0 / 8.7, 24 of 100000 cut into 256 / 512 215 / 220, 192 of up to 2000 in
  // e4m3 22.9 / 21.0, 2048 of up to 1000 112 / 100 and 81 / 58, 1280 of 34 21.5 / 13.2, 2048 of up to 4096 395 / 390.)
  s.waves = !only_short || tiles[0] * kv_heads > 128 ? 4 : kAttnWaves;
  s.slots = a.solo ? 2048 : only_short && s.waves == 4 ? 512 : 256, l.waves = 4;
  if (a.solo) s.rounds = 2, s.min_blocks = 4;                 // (a wavefront takes 6 us for four blocks)
  for (int which = 0; which < kAttnLists; which++) {
    AttnList& x = a.list[which];
    // (as the kernel cuts them: into the shares of whole rounds of workgroups; a cut tile has two at least)
    const long units = tiles[which] * kv_heads, whole = units < (long)x.rounds * x.slots ? units : (long)x.rounds * x.slots;
    long shares = (whole + x.slots - 1) / x.slots * x.slots / kv_heads;
    if (sharing > 0 && which == 1 && most > a.short_rows && tiles[1] > 0) shares = std::max(shares, (long)kAttnRounds * x.slots / kv_heads);
    x.max_joins = (int)(tiles[which] < shares / 2 ? tiles[which] : shares / 2);
    x.max_parts = (int)(tiles[which] > 0 ? shares : 0);
    x.max_items = (int)(tiles[which] > shares ? tiles[which] : shares);
    // (of a group tiles are shares, cut or not.  Of the long list those are few, whatever prompts there are beside them: 8 sequences of 64 heads over 8 with 32768 new tokens have
    // 80 MB of scratch, 70 without groups; a place for every row, twice, was 2.2 GB.)
    if (sharing > 0 && which != 1) x.max_joins = (int)tiles[which], x.max_parts = x.max_items;
    if (sharing > 0 && which == 1) x.max_parts = (int)std::max(shares, kept), x.max_joins = (int)std::min(tiles[1], joined + x.max_parts / 2);
  }
  long at = sharing > 0 ? 16 : 8;
  for (int which = 0; which < kAttnLists; which++) {
    AttnList& x = a.list[which];
    x.items = at, at += 8L * x.max_items;
    x.joins = at, at += 8L * x.max_joins;
    if (sharing > 0) x.prefixes = at, at += 2L * tiles[which];
  }
  a.map = at;
  if (sharing > 0) at += a.shared_rows / a.group;
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
  int start, n, kv, from;                                // from: where its own part of the context begins, a whole number of blocks
};
// the tokens of the cache that some row of a tile sees, its beginning on a whole block
__device__ __forceinline__ void attn_range(const AttnSeq& s, int tile, int rows, const AttnLayout& a, int* lo, int* hi) {
  const uint32_t row = (uint32_t)tile * rows;            // (tokens times heads of a group are below 2^31)
  const int t0 = (int)(row / (uint32_t)a.group), t1 = min(s.n - 1, (int)((row + rows - 1) / (uint32_t)a.group));
  const long before = (long)s.kv - s.n;
  *hi = a.causal ? (int)max(0L, before + t1 + 1) : s.kv;
  *lo = a.window > 0 ? (int)max(0L, before + t0 - a.window + 1) / kAttnBlock * kAttnBlock : s.from;
  *lo = min(*lo, *hi / kAttnBlock * kAttnBlock);
}

// What is known of groups, in LDS.  Of the sequences behind n_seqs, n_seqs + 1 + g is the prefix of group g.
template <bool SHARED>
struct AttnGroups {
  static constexpr int kSize = SHARED ? kAttnMaxGroups + 1 : 1;
  int start[kSize], first[kSize], least[kSize], few[kSize], tokens[kSize];      // of the sequences that share; few: those of up to kAttnSharedRows rows
  int mixed[kSize];                                      // prompts among the group's sequences
  int more;                                              // rows of sequences that share if they fit
  int listed;                                            // whether some prefix's tokens are in the plan's list
  unsigned long long saved, rows;                        // blocks that are not read again, rows to join
  int prompts, wide;                                     // tiles of 128 rows: of sequences that share nothing, of prefixes
  int own;                                               // blocks of a head that the sequences' own parts have
  int longest;
  int home[SHARED ? kAttnMaxSeqs : 1];                   // the group that a sequence shares with, -1: none
  int place[SHARED ? kAttnMaxSeqs : 1];                  // of its tokens among those that are listed
};

// grid 1, block kAttnPlanThreads, or 192 of groups
template <bool SHARED>
__global__ __launch_bounds__(SHARED ? 192 : kAttnPlanThreads) void attention_plan_kernel(const int* q_starts, const int* kv_lens, const int* group_starts, const int* prefix_lens,
                                                                          AttnLayout a, int* plan) {
  __shared__ int start[kAttnMaxSeqs + 1], count[kAttnMaxSeqs + 1], context[kAttnMaxSeqs + 1];
  constexpr int kThreads = SHARED ? 192 : kAttnPlanThreads, kLists = kThreads / 64;
  __shared__ int tiles_ahead[kLists][kAttnMaxSeqs + 1];  // of each sequence, in each list
  __shared__ int order[kLists][kAttnSorted];
  __shared__ int crossed[kLists];
  __shared__ AttnGroups<SHARED> groups;
  bool back = false;                                     // an offset below the one ahead of it
  for (int b = threadIdx.x; b <= a.n_seqs; b += kThreads) {
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
  for (int w = 0; w < kLists; w++) mend |= crossed[w] != 0;
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
  bool pays = false;
  const int last = SHARED ? a.n_seqs + a.n_groups : a.n_seqs;      // of the sequences, the tokens behind them and the prefixes among them
  if constexpr (SHARED) {
    bool unordered = false;
    for (int g = threadIdx.x; g <= a.n_groups; g += kThreads) {
      const int at = max(0, min(group_starts[g], a.n_seqs));
      groups.start[g] = at, groups.least[g] = 0x7e000000, groups.few[g] = groups.tokens[g] = groups.mixed[g] = 0, groups.first[g] = 0x7fffffff;
      if (g > 0) unordered |= at < max(0, min(group_starts[g - 1], a.n_seqs));
    }
    const bool any_unordered = __any(unordered);
    if (threadIdx.x == 0) groups.saved = groups.rows = 0, groups.longest = groups.own = groups.listed = groups.prompts = groups.wide = groups.more = 0;
    __syncthreads();                                     // (`crossed` has been read)
    if ((threadIdx.x & 63) == 0) crossed[threadIdx.x >> 6] = any_unordered;
    __syncthreads();
    if ((crossed[0] | crossed[1] | crossed[kLists - 1]) != 0) {
      if (threadIdx.x == 0)
        for (int g = 1; g <= a.n_groups; g++) groups.start[g] = max(groups.start[g], groups.start[g - 1]);
      __syncthreads();
    }
    for (int b = threadIdx.x; b < a.n_seqs; b += kThreads) {
      int lo = -1, hi = a.n_groups;                      // the last group that starts at or ahead of sequence b
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (groups.start[mid] <= b) lo = mid; else hi = mid - 1;
      }
      if (lo == a.n_groups || count[b] == 0) lo = -1;    // behind the last
      groups.home[b] = lo;
      const long rows = (long)count[b] * a.group;
      if (lo >= 0 && rows > kAttnSharedRows && rows <= kAttnMostRows) atomicAdd(&groups.more, (int)rows);
    }
    __syncthreads();
    const int most_rows = groups.more <= kAttnMoreRows ? kAttnMostRows : kAttnSharedRows;
    for (int b = threadIdx.x; b < a.n_seqs; b += kThreads) {
      const int home = groups.home[b];
      const long rows = (long)count[b] * a.group;
      if (home >= 0 && rows <= most_rows) {
        atomicMin(&groups.least[home], a.causal ? context[b] - count[b] : context[b]);
        atomicMin(&groups.first[home], b);
        atomicAdd(&groups.tokens[home], count[b]);
        if (rows <= kAttnSharedRows) atomicAdd(&groups.few[home], 1);
      } else {
        if (home >= 0) groups.home[b] = -1, groups.mixed[home] = 1;
        if (rows > a.short_rows) atomicAdd(&groups.prompts, (int)((rows + kAttnTileRows - 1) / kAttnTileRows));
      }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < a.n_groups; g += kThreads) {
      // (a window hides of the prefix from each row what it hides; nothing is shared then)
      int prefix = groups.few[g] < 2 || a.window > 0 ? 0 : min(prefix_lens[g], groups.least[g]);
      prefix = max(prefix, 0) / kAttnBlock * kAttnBlock;
      const int b = a.n_seqs + 1 + g;
      start[b] = count[b] = 0, context[b] = prefix;
      if (prefix > 0) {
        start[b] = start[groups.first[g]], count[b] = groups.tokens[g];
        if (groups.mixed[g]) {
          int end = groups.start[g + 1] - 1;             // the last that shares
          while (groups.home[end] != g) end--;
          if (start[end] + count[end] - start[b] != count[b]) start[b] = -1, groups.listed = 1;      // (not adjacent: placed below)
        }
        atomicAdd(&groups.saved, (unsigned long long)(groups.few[g] - 1) * (prefix / kAttnBlock) * a.kv_heads);
        atomicAdd(&groups.rows, (unsigned long long)count[b] * a.group * a.kv_heads);
        atomicMax(&groups.longest, prefix / kAttnBlock);
        if (count[b] * a.group > kAttnPrefixRows || start[b] < 0) atomicAdd(&groups.wide, (count[b] * a.group + kAttnTileRows - 1) / kAttnTileRows);
      }
    }
    __syncthreads();
    // Whether it pays.  A block that is read again comes from the caches, 2 to 3 ns of the whole chip; sharing takes a second walk and a join of every row.  On 196 batches of 2 to
    // 128 single tokens behind 128 to 8192 shared ones, over 8 and 32 heads of the cache, the choice is 0.4 % behind the better of both on average, 19 % at most: 64 requests of
    // 64 heads behind 512 tokens 13.9 us each for itself and 19.0 shared, behind 2048 33.7 and 26.0, behind 8192 124 and 48.
    pays = 10 * groups.saved >= 40000 + 6 * groups.rows || (groups.saved > 0 && groups.longest >= 12 && a.n_seqs * a.kv_heads <= 256);
    // Not where prompts fill whole rounds of workgroups and the prefixes' tiles would begin another: 64 requests and a prompt of 2048 behind 8192 774 us, shared 885; 32 and one of 1000 behind
    // 4096 219 and 260.
    const uint32_t slots = a.list[1].slots, prompts = (uint32_t)groups.prompts * a.kv_heads, with = prompts + (uint32_t)groups.wide * a.kv_heads;      // (below 2^31)
    if (4L * prompts >= 3L * with && (with + slots - 1) / slots > (prompts + slots - 1) / slots) pays = false;
    if (!pays)
      for (int g = threadIdx.x; g < a.n_groups; g += kThreads) count[a.n_seqs + 1 + g] = context[a.n_seqs + 1 + g] = 0;
    __syncthreads();
    if (pays && groups.listed) {
      if (threadIdx.x < 64) {
        int listed = 0, all;
        for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
          const int b = b0 + threadIdx.x, home = b < a.n_seqs ? groups.home[b] : -1;
          const int before = attn_scan(home >= 0 && start[a.n_seqs + 1 + home] < 0 ? count[b] : 0, &all);
          if (b < a.n_seqs) groups.place[b] = listed + before;
          listed += all;
        }
      }
      __syncthreads();
      for (int b = threadIdx.x; b < a.n_seqs; b += kThreads)
        if (groups.home[b] >= 0 && start[a.n_seqs + 1 + groups.home[b]] < 0)
          for (int i = 0; i < count[b]; i++) plan[a.map + groups.place[b] + i] = start[b] + i;
      __syncthreads();
      // (what attn_token reads: below zero, the plan's index)
      for (int g = threadIdx.x; g < a.n_groups; g += kThreads)
        if (start[a.n_seqs + 1 + g] < 0) start[a.n_seqs + 1 + g] = ~(int)(a.map + groups.place[groups.first[g]]);
    }
    if (pays) {
      int own = 0, all;
      for (int b = threadIdx.x; b < a.n_seqs; b += kThreads)
        if (count[b] > 0) own += min((context[b] - (groups.home[b] >= 0 ? context[a.n_seqs + 1 + groups.home[b]] : 0)) / kAttnBlock, 1 << 18);
      attn_scan(own, &all);
      if ((threadIdx.x & 63) == 0) atomicAdd(&groups.own, all);      // (read behind the next barrier)
    }
  }
  const int which = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const AttnList& l = a.list[which];
  if (l.max_items == 0) {
    if (lane < 2) plan[2 * which + lane] = 0;
    if (SHARED && lane == 0) plan[6 + which] = 0;
    if constexpr (SHARED) __syncthreads();
    return;
  }
  auto from_of = [&](int b) { return SHARED && b < a.n_seqs && groups.home[b] >= 0 ? context[a.n_seqs + 1 + groups.home[b]] : 0; };
  auto list_of = [&](int b, long rows) {                         // of sequence b, the tokens behind the last or a prefix
    if (SHARED && b > a.n_seqs) return rows <= kAttnPrefixRows && start[b] >= 0 ? 2 : 1;      // (tiles only take their tokens from a list)
    if (SHARED && b < a.n_seqs && rows <= a.short_rows && context[b] - from_of(b) > kAttnOwnBlocks * kAttnBlock) return 2;
    return rows <= a.short_rows ? 0 : 1;
  };
  int* ahead = tiles_ahead[which];
  int tiles = 0;
  for (int b0 = 0; b0 <= last; b0 += 64) {
    const int b = b0 + lane;
    int mine = 0;
    if (b <= last) {
      const long rows = (long)count[b] * a.group;
      if (rows > 0 && list_of(b, rows) == which) mine = (int)((rows + l.rows - 1) / l.rows);
    }
    int all;
    const int before = attn_scan(mine, &all);
    if (b <= last) ahead[b] = tiles + before;
    tiles += all;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");        // (the wavefront's own list: its lanes run together)
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  if constexpr (SHARED) __syncthreads();                         // (a tile's prefix may be in the other list)
  struct Tile {
    int seq, tile, lo, hi, blocks, home;                         // home: the sequence that is its prefix, -1: none, -2: a prefix itself
    AttnSeq s;
  };
  auto at = [&](int i) {
    int lo = 0, hi = last;                                       // the last sequence that starts at or ahead of tile i
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (ahead[mid] <= i) lo = mid; else hi = mid - 1;
    }
    Tile t;
    t.seq = lo, t.tile = i - ahead[lo], t.s = {start[lo], count[lo], context[lo], 0};
    if (SHARED && lo > a.n_seqs) {
      t.seq = groups.first[lo - a.n_seqs - 1], t.s.kv += t.s.n;  // (as if the new tokens came behind it: all of them see all of it)
      t.lo = 0, t.hi = context[lo], t.home = -2;
    } else {
      t.home = -1;
      if (SHARED && lo < a.n_seqs && groups.home[lo] >= 0 && context[a.n_seqs + 1 + groups.home[lo]] > 0) {
        t.home = a.n_seqs + 1 + groups.home[lo];
        t.s.from = context[t.home];
      }
      attn_range(t.s, t.tile, l.rows, a, &t.lo, &t.hi);
    }
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
    int most = (int)((units + l.slots - 1) / l.slots * l.slots / a.kv_heads);              // shares of one head
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
    if (pays && which > 0 && units <= l.slots / 2 && (long)total * a.kv_heads <= kAttnHalf * l.slots / 2) {
      // Short walks leave slots to the own parts, and fewer results to join: half the slots.  Tiles: the more, the longer their walks and the less there is beside them.  (us with 3, 4, 5, 6 and
      // 8 eighths of them: 64 requests of 64 heads over 8 behind 8200 tokens 61, 55, 51, 52, 61, of 32 + 32 heads 85, 93, 94, 95, 101; on 294 such batches of 32 to 128 requests 2.3 % behind
      // the best of them on average, half the slots 5.2 %.)
      const long walk = (long)total * a.kv_heads;
      const long beside = SHARED ? 2L * groups.own * a.kv_heads : 0;
      int eighths = 4;
      if (which == 1) {
        const bool some = walk * 2 >= 5L * l.slots / 2;
        eighths = (walk >= 9L * l.slots / 2 ? 6 : some ? 5 : 3) - (beside >= walk) - (some && beside >= 5 * walk);
      }
      most = l.slots * eighths / 8 / a.kv_heads;
    }
    int longest = 0;
    if constexpr (SHARED) {
#pragma unroll
      for (int k = 0; k < kAttnSorted / 64; k++) longest = max(longest, mine[k]);
#pragma unroll
      for (int d = 32; d > 0; d /= 2) longest = max(longest, __shfl_xor(longest, d));
    }
    auto cut_into = [&](int shares) {
      int blocks = max(!SHARED || pays || which == 0 ? l.min_blocks : which == 1 ? kAttnTileBlocks : kAttnRowBlocks, (total + shares - 1) / max(shares, 1));
      if (pays) blocks = max(blocks, (longest + 15) / 16);       // (a row's shares are joined: sixteen at most for this)
      while (blocks <= total && sum_of([&](int n) { return max(1, (n + blocks - 1) / blocks); }) > shares) blocks += (blocks + 7) / 8;
      return blocks;
    };
    share = cut_into(most);
    if (SHARED && !pays && which == 1 && tiles <= kAttnSorted) {  // (a batch without groups keeps its cut, and with it its bits)
      int rounds = max(1, most * a.kv_heads / l.slots), least = rounds * (min(share, longest) + kAttnShareBlocks);
      while (++rounds <= kAttnRounds && rounds * l.slots / a.kv_heads <= l.max_parts) {
        const int other = cut_into(rounds * l.slots / a.kv_heads), cost = rounds * (min(other, longest) + kAttnShareBlocks);
        if (cost < least) least = cost, share = other;
      }
    }
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
  int n_items = 0, n_joins = 0, n_parts = 0, fullest = 0;        // fullest: rows of a tile that is joined, at most
  int end_items = l.max_items, end_joins = l.max_joins;          // (all have a place: the cut leaves no more shares than the host has counted)
  for (int i0 = 0; i0 < tiles; i0 += 64) {
    // (of long lists a sequence's last tile, its longest, first)
    const int i = i0 + lane >= tiles ? -1 : tiles <= kAttnSorted ? order[which][i0 + lane] : tiles - 1 - (i0 + lane);
    int splits = 0, per = 0;
    Tile t = {};
    t.home = -1;
    if (i >= 0) {
      t = at(i);
      splits = max(1, (int)(((long)t.blocks + share - 1) / share));
      per = (t.blocks + splits - 1) / splits;
      splits = per > 0 ? max(1, (t.blocks + per - 1) / per) : 1;
    }
    int all_items, all_joins, all_parts;
    const int item = n_items + attn_scan(splits, &all_items);
    const bool cut = splits > 1 || (SHARED && i >= 0 && t.home != -1), joins = cut && t.home != -2;
    const int join = n_joins + attn_scan(joins, &all_joins);
    const int part = n_parts + attn_scan(cut ? splits : 0, &all_parts);
    if (i >= 0 && (item + splits > l.max_items || (joins && join >= l.max_joins) || (cut && part + splits > l.max_parts))) {
      end_items = min(end_items, item), end_joins = min(end_joins, join);
    } else if (i >= 0) {
      AttnItem* out = reinterpret_cast<AttnItem*>(plan + l.items) + item;
      for (int p = 0; p < splits; p++)
        out[p] = AttnItem{t.seq, t.s.start, t.s.n, t.s.kv, t.tile, t.lo + p * per * kAttnBlock, splits == 1 ? t.hi : min(t.hi, t.lo + (p + 1) * per * kAttnBlock),
                          cut ? part + p : -1};
      AttnJoin j = {t.s.start, t.s.n, t.tile, part, splits, -1, 0, 0};
      if (SHARED && t.home > 0) {
        j.prefix_list = list_of(t.home, (long)count[t.home] * a.group);
        const int ahead_of = start[t.home] < 0 ? groups.place[t.seq] - groups.place[groups.first[t.home - a.n_seqs - 1]] : t.s.start - start[t.home];
        j.prefix_tile = tiles_ahead[j.prefix_list][t.home], j.prefix_row = ahead_of * a.group;
      }
      if (SHARED && joins) fullest = max(fullest, min(l.rows, t.s.n * a.group - t.tile * l.rows));
      if (joins) reinterpret_cast<AttnJoin*>(plan + l.joins)[join] = j;
      if (SHARED && t.home == -2) plan[l.prefixes + 2L * i] = part, plan[l.prefixes + 2L * i + 1] = splits;
    }
    n_items += all_items, n_joins += all_joins, n_parts += all_parts;
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) end_items = min(end_items, __shfl_xor(end_items, d)), end_joins = min(end_joins, __shfl_xor(end_joins, d));
  if (lane == 0) plan[2 * which] = min(n_items, end_items), plan[2 * which + 1] = min(n_joins, end_joins);
  if constexpr (SHARED) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) fullest = max(fullest, __shfl_xor(fullest, d));
    if (lane == 0) plan[6 + which] = fullest;
  }
}

}  // namespace triteia_hip
