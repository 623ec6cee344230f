// Attention of new tokens over a paged cache: out = softmax(scale q K^T, masked) V, per head, on a plan's items (attention_plan.hip.h).
//
// Pages [n_pages, kv_heads, page, D] of the activations' type, or of int8 / e4m3 codes with a 32-bit scale per row.  Row r of a tile is
// token r / group of its sequence and head r % group of the cache head's group; with causal its last token is the sequence's
// newest, a window keeps the last `window` tokens.  Both kernels work on the transposed product:
//   S^T = K Q^T        an MFMA with tokens of the cache down and rows across, so a lane holds scores of ONE row and the softmax needs
//                      one or two lane exchanges;
//   O^T = V^T P^T      whose operand P^T is, in the accumulator's own layout, what the lane holds already: the order of the tokens inside an
//                      MFMA's K is free as long as V has the same, and ds_read_b64_tr_b16 (_b8) takes four (eight) rows of any addresses and
//                      hands a lane one column of them.  P never leaves the registers.
// Scores, running maxima and sums and the output's sums are 32 bits; P is rounded once to the activations' type for the MFMA.  The maximum is
// a reference that is only moved (and the sums rescaled) when a weight would pass 2^kHigh; it is put where the largest weight is 2^kLow.  fp16 ends at 2^16 and
// loses what is below 2^-25, so its largest weight stands at 2^7 to 2^15 and one of 2^-24 of it keeps 8 bits; beside a largest of 1, ten thousand of 2^-26
// counted in the sum and not in the output.  bf16 has the exponents of 32 bits.  Over 8-bit caches P takes V's scales in (kept out of V, whose rounding would
// grow), and fp16's range is kept by the row's largest weight times scale, `peak`, in the same way (attn_shift): by the largest scale, a value far above the others
// with a weight of next to nothing took their bits.
// Masked scores are -infinity ahead of the maximum; a row that sees nothing has a sum of zero and gives zeros.  What is masked for some rows of
// a tile and holds an infinity or a NaN in V must not reach those rows by 0 * inf: blocks on such an edge enter LDS without them (attn_clean),
// and the rows that see them get them added one by one (attn_strange).
#pragma once
#include "attention_plan.hip.h"
#include "kv_cache.hip.h"

namespace triteia_hip {

typedef float attn_f4 __attribute__((ext_vector_type(4)));
typedef float attn_f16 __attribute__((ext_vector_type(16)));
typedef short attn_s4 __attribute__((ext_vector_type(4)));
typedef int attn_i2 __attribute__((ext_vector_type(2)));

constexpr float kAttnNone = -3e38f;     // the maximum of nothing: below every score that is a number, but for the last eighth of their range

struct AttendArgs {
  const void* q;
  long q_token, q_head;
  void* out;                            // [tokens, heads, D]
  CachePart ck, cv;
  const int* pages;
  long pages_seq;                       // stride
  int n_pages, table_width, page_shift;
  int held, joined;                     // tokens that a row of the table holds; whether a launch behind joins shares
  int group, kv_heads, causal, window;
  float scale_log2;                     // scale * log2(e)
  const int* plan;
  AttnList list[kAttnLists];
  float *part_o[kAttnLists], *part_ml[kAttnLists];        // of each list: [parts][kv_heads][rows][D], [parts][kv_heads][rows][2]
};

// The largest over lanes 32 apart, or 16 and 32 apart, in all of them: whole rows of lanes trade places on the vector ALU.
__device__ __forceinline__ float attn_max32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float attn_max16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t lo = r[0], hi = r[1];
  return attn_max32(fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)));
}

template <class T>
struct AttnMma;
template <>
struct AttnMma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7c00;
  static constexpr float kLow = 7.f, kHigh = 15.f;
  static __device__ __forceinline__ attn_f4 m16(v8 a, v8 b, attn_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ attn_f16 m32(v8 a, v8 b, attn_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct AttnMma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7f80;
  static constexpr float kLow = 0.f, kHigh = 8.f;
  static __device__ __forceinline__ attn_f4 m16(v8 a, v8 b, attn_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ attn_f16 m32(v8 a, v8 b, attn_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// 16 bytes of V without their infinities and NaNs; whether there were any.
template <class T, int KIND>
__device__ __forceinline__ bool attn_clean(kv_uint4* v) {
  uint32_t found = 0;
  if constexpr (KIND != kCacheInt8) {
    // magnitudes from the least that is no number on carry into the sign's place (e4m3 has one NaN and no infinity)
    constexpr uint32_t magnitude = KIND == kCacheSame ? 0x7fff7fffu : 0x7f7f7f7fu, sign = ~magnitude;
    constexpr uint32_t carry = KIND == kCacheSame ? (0x8000u - AttnMma<T>::kInf) * 0x00010001u : 0x01010101u;
    constexpr int bits = KIND == kCacheSame ? 15 : 7;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t odd = (((*v)[i] & magnitude) + carry) & sign;
      (*v)[i] &= ~(odd | (odd - (odd >> bits)));
      found |= odd;
    }
  }
  return found != 0;
}

// What attn_clean took out, for rows that see it: V's infinities and NaNs among four elements of a token's row, zeros for all that is finite.
template <class T, int KIND>
__device__ __forceinline__ attn_f4 attn_strange(const CachePart& c, long page, int head, int slot, int d) {
  attn_f4 x = {0.f, 0.f, 0.f, 0.f};
  const long at = page * c.page + head * c.head + slot * c.slot + d;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (KIND == kCacheSame) {
      const float v = (float)static_cast<const T*>(c.data)[at + j];
      if (!(__builtin_fabsf(v) < __builtin_inff())) x[j] = v;
    } else if constexpr (KIND == kCacheFp8) {
      if ((static_cast<const uint8_t*>(c.data)[at + j] & 0x7f) == 0x7f) x[j] = __builtin_nanf("");
    }
  }
  return x;
}

// 8 codes as 8 values of the activations' type, exactly
template <class T, int KIND>
__device__ __forceinline__ kv8<T> attn_values(kv_uint2 c) {
  kv8<T> out;
  typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; i++) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      t2 pair;
      if constexpr (KIND == kCacheFp8) {
        if constexpr (__is_same(T, _Float16)) pair = j ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false);
        else pair = j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, false);
      } else if constexpr (__is_same(T, _Float16)) {
        // (code + 128 in the low bits of 1024, and 1152 taken off)
        const uint32_t w = __builtin_amdgcn_perm(0x64646464u, c[i] ^ 0x80808080u, j ? 0x04030402u : 0x04010400u);
        pair = __builtin_bit_cast(t2, w) - t2{(T)1152.f, (T)1152.f};
      } else {
        pair = t2{(T)(float)(int)(int8_t)(c[i] >> (16 * j)), (T)(float)(int)(int8_t)(c[i] >> (16 * j + 8))};
      }
      out[4 * i + 2 * j] = pair.x, out[4 * i + 2 * j + 1] = pair.y;
    }
  }
  return out;
}

template <class T>
__device__ __forceinline__ kv8<T> attn_transposed(const uint8_t* lds, int first, int second) {    // four rows at each
  typedef T t4 __attribute__((ext_vector_type(4)));
  const t4 a = __builtin_bit_cast(t4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn_s4*)(lds + first)));
  const t4 b = __builtin_bit_cast(t4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn_s4*)(lds + second)));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ AttnItem attn_item(const AttendArgs& a, int which, int i) {
  const int* p = a.plan + a.list[which].items + 8L * i;
  return AttnItem{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
}

// the page of a token, kept inside the table and the cache
__device__ __forceinline__ int attn_page(const AttendArgs& a, int seq, int token) {
  const int at = min(token >> a.page_shift, a.table_width - 1);
  return (int)min((uint32_t)a.pages[seq * a.pages_seq + at], (uint32_t)(a.n_pages - 1));
}

// One head's keys or values.  Where the 16 tokens of a group start is the same for all lanes and the base of a buffer; a lane's own offset from there, and
// the offset of the rows of each further request, have 32 bits.  (Added up as 64-bit addresses they were half of the loop's scalar instructions.)
// ONCE: every row is read by one workgroup alone, as a decode step's are, and need not stay in the caches (64 contexts of up to 4096 tokens, 32 heads, 430 us
// without that and 386, 3 of up to 100000 in int8 85.0 and 76.4; tiles of 128 rows, which share them, 335 and 349).
template <int ROWS, bool ONCE>     // rows of a request
struct AttnHeld {
  const uint8_t* head;
  long page;                       // strides in bytes
  uint32_t slot, step, lane;
  __device__ __forceinline__ AttnHeld(const CachePart& c, int h, int size, int row, int piece)
      : head(static_cast<const uint8_t*>(c.data) + h * c.head * size), page(c.page * size), slot((uint32_t)(c.slot * size)), step(ROWS * slot),
        lane(row * slot + 16 * piece) {}
  template <int N>
  __device__ __forceinline__ void read(kv_uint4* to, long p, int first) const {
    const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(head) + p * page + (long)first * slot, 0, 0xffffffffu, 0x00027000);
#pragma unroll
    for (int j = 0; j < N; j++) to[j] = __builtin_bit_cast(kv_uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, lane, j * step, ONCE ? 2 : 0));
  }
};

// The tokens that a lane's row sees of a block, for the branches of blocks on an edge: a value of its own in each, or the compiler takes the comparisons of all
// branches out of them and does them for every block (4 x 500 new tokens behind up to 8200 in e4m3 were 440 us that way, 373 this).
struct AttnSpan {
  int lo, hi;
  __device__ __forceinline__ AttnSpan here() const {
    AttnSpan x = *this;
    asm volatile("" : "+v"(x.lo), "+v"(x.hi));
    return x;
  }
  __device__ __forceinline__ bool hides(int token) const { return token < lo || token >= hi; }
};

// The power of two by which a row's sums and weights move so that its largest weight times scale, which has left 1 .. 2^15, is 2^7 to 2^8 again.  (Exact; the
// reference of scores is a whole number where this is in use, so that less the shift it is exact too, up to attn_far.)  Beyond 2^+-64 fp16's outputs have ended.
__device__ __forceinline__ bool attn_off(float peak) { return peak > 32768.f || (peak < 1.f && peak > 0.f); }
__device__ __forceinline__ int attn_shift(float peak, int now) { return attn_off(peak) ? max(-64, min(64, now + 8 - __builtin_amdgcn_frexp_expf(peak))) - now : 0; }

// A reference so large that its rounding, which a product inside an fma does not share, would pass an exponential's end, or that takes the shift up.
__device__ __forceinline__ bool attn_far(float m) { return __builtin_fabsf(m) > 1048576.f && m > kAttnNone; }

// Which tokens row `r` of a tile sees: lo <= token < hi.  Rows behind the last see all that the tile sees and are not stored.
struct AttnRow {
  int lo, hi, token, head;     // token of the sequence, head of the group
  bool live;
};
__device__ __forceinline__ AttnRow attn_row(const AttendArgs& a, const AttnItem& it, int rows, int r) {
  const uint32_t row = (uint32_t)it.tile * rows + r;       // (tokens times heads of a group are below 2^31)
  AttnRow x;
  x.token = (int)(row / (uint32_t)a.group), x.head = (int)(row - (uint32_t)x.token * a.group);
  x.live = x.token < it.n_tokens;
  const int position = it.kv_len - it.n_tokens + x.token;
  x.hi = x.live && a.causal ? min(position + 1, it.kv_len) : it.kv_len;
  x.lo = x.live && a.window > 0 ? max(0, max(position, 0) - a.window + 1) : 0;      // (a window may be as long as an int is large)
  if (!x.live) x.token = 0, x.head = 0;
  return x;
}

// A token's row of the queries.  LISTED: the item may be a prefix's, whose tokens need not be adjacent: below zero q_start is the complement of where the plan lists them.  (Only tiles
// of 128 rows ask: in the walks of few rows, which wait for their first loads, 96 requests behind six prefixes of 3000 took 80 us with it and 75.5 without.)
template <bool LISTED>
__device__ __forceinline__ int attn_token(const AttendArgs& a, const AttnItem& it, int token) {
  if (LISTED && it.q_start < 0) return a.plan[~it.q_start + token];
  return it.q_start + token;
}

// The plan knows lengths, not the table: an item is held to the tokens that the table has.  Where no context that the table can hold is worth cutting there
// is no launch that joins, and a plan that has cut all the same (for lengths that the table cannot hold) leaves the tile to its first share, which takes
// all of it.  False: nothing is left to do.
__device__ __forceinline__ bool attn_within(const AttendArgs& a, int rows, AttnItem* it) {
  if (it->part >= 0 && !a.joined) {
    if (it->kv_begin != attn_row(a, *it, rows, 0).lo / kAttnBlock * kAttnBlock) return false;
    it->part = -1, it->kv_end = it->kv_len;
  }
  it->kv_end = min(it->kv_end, a.held), it->kv_begin = min(it->kv_begin, it->kv_end);
  return true;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Few rows: a decode step's heads, a handful of tokens.  Bound by the cache's bytes.  A workgroup takes a share of one tile's tokens; each of
// its four or eight wavefronts walks sub-tiles of its own (8 KB of K and 8 KB of V: 32 tokens of 128 elements in 16 bits, 64 in 8) with the next one's whole rows
// on their way in registers and this one's in LDS of its own, so that the loop has no barrier; maxima, sums and outputs are joined once at the end.
// In 8 bits LDS holds the codes and each is converted once, behind its read (ds_read_b64_tr_b8 hands a lane eight tokens of a column).
// Measured: 64 contexts of up to 4096 tokens, 32 heads, fp16 386 us a call (2.53 GB, 6.6 TB/s); 3 of up to 100000 over 8 heads in int8 76 us (402 MB), 7 of them
// the joining launch's; one of 500 8.0 us, of which about 1 are the plan's and 1 the pages' round trip, 1 the first rows', 2 two sub-tiles and 2 the joining.
template <int KIND, int D, int NQ, int WAVES>
struct AttnRowsLds {
  static constexpr int kRowBytes = D * (KIND == kCacheSame ? 2 : 1);
  static constexpr int kSub = KIND != kCacheSame && NQ == 2 ? 32 : 8192 / kRowBytes < 64 ? 8192 / kRowBytes : 64;   // (two tiles of rows fill the registers)
  static constexpr int kTile = kSub * kRowBytes, kRows = 16 * NQ;
  static constexpr int kStride = D + 4;                                      // floats of a row where the wavefronts meet
  static constexpr int kMeet = WAVES / 2 * kRows * kStride * 4;
  alignas(16) uint8_t tiles[WAVES * 2 * kTile > kMeet ? WAVES * 2 * kTile : kMeet];
  float meet_m[WAVES][kRows], meet_l[WAVES][kRows];
  alignas(16) float scales[KIND == kCacheSame ? 1 : WAVES][2][kSub];
};

template <class T, int KIND, int D, int NQ, int WAVES, int LIST = 0>
__device__ __forceinline__ void attend_rows(const AttendArgs& a, int index, int head, AttnRowsLds<KIND, D, NQ, WAVES>& shared) {
  using M = AttnMma<T>;
  using v8 = typename M::v8;
  using Lds = AttnRowsLds<KIND, D, NQ, WAVES>;
  constexpr int kRowBytes = Lds::kRowBytes, kChunks = kRowBytes / 16, kSub = Lds::kSub, kTile = Lds::kTile, kRows = Lds::kRows, kStride = Lds::kStride;
  constexpr int kLoads = kSub * kChunks / 64, kLoadRows = 64 / kChunks;     // requests of a sub-tile, rows of each
  constexpr int kGroups = kSub / 16, kGroupLoads = kLoads / kGroups;
  constexpr int kKeyRows = 256 / kRowBytes;
  uint8_t* lds = shared.tiles;
  auto& meet_m = shared.meet_m;
  auto& meet_l = shared.meet_l;
  auto& scales = shared.scales;
  AttnItem it = attn_item(a, LIST, index);           // (requested together with the number of items)
  if (index >= a.plan[2 * LIST] || !attn_within(a, kRows, &it)) return;
  const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, h = lane >> 4;
  uint8_t* lds_k = lds + wave * 2 * kTile;
  uint8_t* lds_v = lds_k + kTile;

  const int n_sub = (it.kv_end - it.kv_begin + kSub - 1) / kSub;
  kv_uint4 rk[kLoads], rv[kLoads];
  float ks = 0.f, vs = 0.f;                 // scales of token `lane` of the sub-tile
  const int load_row = lane / kChunks, load_chunk = lane % kChunks;
  const int page_mask = (1 << a.page_shift) - 1;
  const AttnHeld<kLoadRows, true> held_k(a.ck, head, kRowBytes / D, load_row, load_chunk), held_v(a.cv, head, kRowBytes / D, load_row, load_chunk);
  const float *scale_k = a.ck.scale + head * a.ck.scale_head, *scale_v = a.cv.scale + head * a.cv.scale_head;
  // A lane fetches the page of one 16-token group of the wavefront's next sub-tiles: kIds sub-tiles' pages are one request, a request ahead.
  constexpr int kIds = 64 / kGroups;
  auto pages_from = [&](int i) {
    const long token = it.kv_begin + (wave + (long)WAVES * (i + lane / kGroups)) * kSub + 16 * (lane % kGroups);
    return attn_page(a, it.seq, (int)min(token, (long)it.kv_end - 1));
  };
  int ids = n_sub > wave ? pages_from(0) : 0, next_ids = n_sub > wave + WAVES * kIds ? pages_from(kIds) : 0;
  auto request = [&](int i) {                // the wavefront's i-th sub-tile
    const int t0 = it.kv_begin + (wave + WAVES * i) * kSub;
    if (i > 0 && i % kIds == 0) {
      ids = next_ids;
      if (wave + WAVES * (i + kIds) < n_sub) next_ids = pages_from(i + kIds);
    }
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
      const long page = __builtin_amdgcn_readlane(ids, i % kIds * kGroups + g);
      const int slot = min(t0 + 16 * g, (it.kv_end - 1) & ~15) & page_mask;
      held_k.template read<kGroupLoads>(rk + g * kGroupLoads, page, slot);
      held_v.template read<kGroupLoads>(rv + g * kGroupLoads, page, slot);
    }
    if constexpr (KIND != kCacheSame) {
      const long page = __shfl(ids, i % kIds * kGroups + lane / 16);
      const int slot = (min(t0 + 16 * (lane / 16), (it.kv_end - 1) & ~15) & page_mask) + col;
      if (lane < kSub) ks = scale_k[page * a.ck.scale_page + slot], vs = scale_v[page * a.cv.scale_page + slot];
    }
  };
  auto key_of = [](int row) { return (row / kKeyRows) & (kChunks - 1); };
  auto key_of_v = [](int row) {
    return KIND == kCacheSame ? (row / kKeyRows << 1) & (kChunks - 1) : ((row / kKeyRows) & (kChunks / 2 - 1)) | ((row >> 4) & 1) * (kChunks / 2);
  };

  if (wave < n_sub) request(0);
  v8 qf[NQ][D / 32];
  int row_lo[NQ], row_hi[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const AttnRow r = attn_row(a, it, kRows, 16 * n + col);
    row_lo[n] = r.lo, row_hi[n] = r.hi;
    const T* src = static_cast<const T*>(a.q) + (it.q_start + r.token) * a.q_token + (head * a.group + r.head) * a.q_head;
#pragma unroll
    for (int s = 0; s < D / 32; s++) {
      const int d = KIND == kCacheSame ? 32 * s + 8 * h : 64 * (s / 2) + 16 * h + 8 * (s % 2);
      qf[n][s] = r.live ? *reinterpret_cast<const v8*>(src + d) : v8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  // the tile's masks: no token ahead of `all_lo` or from `all_hi` on is hidden from some of its rows only
  const AttnRow first = attn_row(a, it, kRows, 0);
  const int last_row = min(kRows, it.n_tokens * a.group - it.tile * kRows) - 1;
  const AttnRow last = attn_row(a, it, kRows, last_row);
  const int all_lo = last.lo, all_hi = first.hi;

  attn_f4 o[NQ][D / 16];
  constexpr bool kNormed = KIND != kCacheSame && __is_same(T, _Float16);
  float m[NQ], l[NQ], peak[NQ];              // l, o and peak are times 2^shift
  int shift[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    m[n] = kAttnNone, l[n] = 0.f, peak[n] = 0.f, shift[n] = 0;
#pragma unroll
    for (int d = 0; d < D / 16; d++) o[n][d] = attn_f4{0.f, 0.f, 0.f, 0.f};
  }
  for (int sub = wave; sub < n_sub; sub += WAVES) {
    const int t0 = it.kv_begin + sub * kSub;
    if (t0 + kSub > it.kv_end) {             // tokens behind the last: whatever the page holds there must not meet a zero of P
#pragma unroll
      for (int j = 0; j < kLoads; j++)
        if (t0 + j * kLoadRows + load_row >= it.kv_end) rv[j] = kv_uint4{0, 0, 0, 0};
    }
    // a block with tokens that some of its rows see and others do not
    const bool edge = t0 < all_lo || t0 + kSub > min(all_hi, it.kv_end);
    bool strange = false;
    if (t0 < all_lo || (t0 + kSub > all_hi && all_hi < it.kv_end)) {
#pragma unroll
      for (int j = 0; j < kLoads; j++) strange |= attn_clean<T, KIND>(&rv[j]);
      strange = __any(strange);
    }
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int row = j * kLoadRows + load_row;
      *reinterpret_cast<kv_uint4*>(lds_k + row * kRowBytes + (load_chunk ^ key_of(row)) * 16) = rk[j];
      *reinterpret_cast<kv_uint4*>(lds_v + row * kRowBytes + (load_chunk ^ key_of_v(row)) * 16) = rv[j];
    }
    if constexpr (KIND != kCacheSame) {
      if (lane < kSub) scales[wave][0][lane] = ks * a.scale_log2, scales[wave][1][lane] = vs;
    }
    if (sub + WAVES < n_sub) request((sub - wave) / WAVES + 1);

    attn_f4 s[NQ][kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
#pragma unroll
      for (int n = 0; n < NQ; n++) s[n][g] = attn_f4{0.f, 0.f, 0.f, 0.f};
      const int row = 16 * g + col;
      if constexpr (KIND == kCacheSame) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const v8 k = *reinterpret_cast<const v8*>(lds_k + row * kRowBytes + ((4 * i + h) ^ key_of(row)) * 16);
#pragma unroll
          for (int n = 0; n < NQ; n++) s[n][g] = M::m16(k, qf[n][i], s[n][g]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
          const kv_uint4 c = *reinterpret_cast<const kv_uint4*>(lds_k + row * kRowBytes + ((4 * i + h) ^ key_of(row)) * 16);
          const v8 k0 = attn_values<T, KIND>(kv_uint2{c[0], c[1]}), k1 = attn_values<T, KIND>(kv_uint2{c[2], c[3]});
#pragma unroll
          for (int n = 0; n < NQ; n++) s[n][g] = M::m16(k1, qf[n][2 * i + 1], M::m16(k0, qf[n][2 * i], s[n][g]));
        }
      }
    }
    v8 p[NQ][kSub / 32];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      float top = kAttnNone;
#pragma unroll
      for (int g = 0; g < kGroups; g++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[n][g][j] *= KIND == kCacheSame ? a.scale_log2 : scales[wave][0][16 * g + 4 * h + j];
          top = fmaxf(top, s[n][g][j]);
        }
      const AttnSpan span = {row_lo[n] - t0 - 4 * h, min(row_hi[n], it.kv_end) - t0 - 4 * h};
      if (edge) {
        const AttnSpan seen = span.here();
        top = kAttnNone;
#pragma unroll
        for (int g = 0; g < kGroups; g++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            s[n][g][j] = seen.hides(16 * g + j) ? -__builtin_inff() : s[n][g][j];
            top = fmaxf(top, s[n][g][j]);
          }
      }
      top = attn_max16(top);
      if (__any(top > m[n] + M::kHigh)) {
        const float low = top - M::kLow, next = fmaxf(m[n], kNormed ? __builtin_floorf(low) : low), f = __builtin_amdgcn_exp2f(m[n] - next);
        l[n] *= f, peak[n] *= f, m[n] = next;
#pragma unroll
        for (int d = 0; d < D / 16; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[n][d][j] *= f;
      }
      float under = kNormed ? m[n] - (float)shift[n] : m[n];
      if constexpr (kNormed) {
        const bool far = attn_far(m[n]);
        if (__any(far)) {
#pragma unroll
          for (int g = 0; g < kGroups; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[n][g][j] -= far ? m[n] : 0.f;
          under = far ? -(float)shift[n] : under;
        }
      }
#pragma unroll
      for (int g = 0; g < kGroups; g++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float e = __builtin_amdgcn_exp2f(s[n][g][j] - under);
          l[n] += e;
          s[n][g][j] = KIND == kCacheSame ? e : e * scales[wave][1][16 * g + 4 * h + j];
        }
      if (KIND != kCacheSame && edge) {              // (a scale may be a NaN)
        const AttnSpan seen = span.here();
#pragma unroll
        for (int g = 0; g < kGroups; g++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[n][g][j] = seen.hides(16 * g + j) ? 0.f : s[n][g][j];
      }
      if constexpr (kNormed) {
        float most = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; g++)
#pragma unroll
          for (int j = 0; j < 4; j++) most = fmaxf(most, __builtin_fabsf(s[n][g][j]));
        peak[n] = fmaxf(peak[n], attn_max16(most));
        if (__any(attn_off(peak[n]))) {
          const int by = attn_shift(peak[n], shift[n]);
          shift[n] += by, peak[n] = __builtin_ldexpf(peak[n], by), l[n] = __builtin_ldexpf(l[n], by);
#pragma unroll
          for (int g = 0; g < kGroups; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[n][g][j] = __builtin_ldexpf(s[n][g][j], by);
#pragma unroll
          for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[n][d][j] = __builtin_ldexpf(o[n][d][j], by);
        }
      }
#pragma unroll
      for (int g = 0; g < kGroups; g++)
#pragma unroll
        for (int j = 0; j < 4; j++) p[n][g / 2][4 * (g % 2) + j] = (T)s[n][g][j];
    }
    auto column = [&](int d, int b) {        // V of 32 tokens from 32 b on, as the MFMA's operand for columns 16 d ..
      if constexpr (KIND == kCacheSame) {
        const int row = 32 * b + 4 * h + col / 4, chunk = 2 * d + (col & 3) / 2, in = 8 * (col & 1);
        return attn_transposed<T>(lds_v, row * kRowBytes + (chunk ^ key_of_v(row)) * 16 + in, (row + 16) * kRowBytes + (chunk ^ key_of_v(row + 16)) * 16 + in);
      } else {
        const int r = col / 2, row = 32 * b + 4 * h + (r & 3) + 16 * (r >> 2);
        const attn_i2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) attn_i2*)(lds_v + row * kRowBytes + (d ^ key_of_v(row)) * 16 + 8 * (col & 1)));
        return attn_values<T, KIND>(kv_uint2{(uint32_t)c.x, (uint32_t)c.y});
      }
    };
#pragma unroll
    for (int d = 0; d < D / 16; d++)
#pragma unroll
      for (int b = 0; b < kSub / 32; b++) {
        const v8 v = column(d, b);
#pragma unroll
        for (int n = 0; n < NQ; n++) o[n][d] = M::m16(v, p[n][b], o[n][d]);
      }
    if (strange) {
#pragma unroll 1
      for (int token = max(t0, 0); token < min(t0 + kSub, it.kv_end); token++) {
        const long page = attn_page(a, it.seq, token);
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
          const attn_f4 x = attn_strange<T, KIND>(a.cv, page, head, token & ((1 << a.page_shift) - 1), 16 * d + 4 * h);
#pragma unroll
          for (int n = 0; n < NQ; n++)
            if (token >= row_lo[n] && token < row_hi[n]) o[n][d] += x;
        }
      }
    }
  }

  if constexpr (WAVES == 1) {                // an item of its own: from the registers
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      const float f = kNormed ? __builtin_ldexpf(1.f, -shift[n]) : 1.f;
      float sum = l[n] * f;
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      const int r = 16 * n + col;
      if (r > last_row) continue;
      const AttnRow row = attn_row(a, it, kRows, r);
      const long at = ((long)it.part * a.kv_heads + head) * (LIST == 2 ? kAttnPrefixRows : kRows) + r;
      T* out = static_cast<T*>(a.out) + ((long)(it.q_start + row.token) * (a.kv_heads * a.group) + head * a.group + row.head) * D;
#pragma unroll
      for (int d = 0; d < D / 16; d++) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const attn_f4 x = o[n][d] * f;
        if (it.part >= 0) *reinterpret_cast<attn_f4*>(a.part_o[LIST] + at * D + 16 * d + 4 * h) = x;
        else *reinterpret_cast<t4*>(out + 16 * d + 4 * h) = sum == 0.f ? t4{0, 0, 0, 0} : t4{(T)(x[0] / sum), (T)(x[1] / sum), (T)(x[2] / sum), (T)(x[3] / sum)};
      }
      if (it.part >= 0 && h == 0) a.part_ml[LIST][2 * at] = m[n], a.part_ml[LIST][2 * at + 1] = sum;
    }
    return;
  }
  // the wavefronts' results: through LDS, the upper half's taken in by the lower half
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    if constexpr (kNormed) l[n] = __builtin_ldexpf(l[n], -shift[n]);
    l[n] += __shfl_xor(l[n], 16);
    l[n] += __shfl_xor(l[n], 32);
    if (h == 0) meet_m[wave][16 * n + col] = m[n], meet_l[wave][16 * n + col] = l[n];
  }
  __syncthreads();
  float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    float top = kAttnNone;
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, meet_m[w][16 * n + col]);
    float f = __builtin_amdgcn_exp2f(m[n] - top);
    if constexpr (kNormed) f = __builtin_ldexpf(f, -shift[n]);
#pragma unroll
    for (int d = 0; d < D / 16; d++)
#pragma unroll
      for (int j = 0; j < 4; j++) o[n][d][j] *= f;
  }
  // (rows that fill half a tile at most, as a decode step's of up to 8 heads do: all at once)
  const bool once = last_row < kRows / 2;
  const int met = once ? WAVES : WAVES / 2, met_rows = once ? kRows / 2 : kRows;
#pragma unroll
  for (int upper = 1; upper >= 0; upper--) {
    if (once ? upper == 1 : (wave >= WAVES / 2) == (upper == 1)) {
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
          attn_f4* to = reinterpret_cast<attn_f4*>(meet + (wave % met * met_rows + 16 * n + col) * kStride + 16 * d + 4 * h);
          if (16 * n + col > last_row) continue;
          if (!upper) o[n][d] += *to;
          *to = o[n][d];
        }
    }
    __syncthreads();
    if (once) break;
  }
  for (int i = threadIdx.x; i < kRows * (D / 4); i += 64 * WAVES) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    if (r > last_row) break;
    float top = kAttnNone, sum = 0.f;
    attn_f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, meet_m[w][r]);
#pragma unroll
    for (int w = 0; w < WAVES; w++) sum += meet_l[w][r] * __builtin_amdgcn_exp2f(meet_m[w][r] - top);
#pragma unroll
    for (int w = 0; w < WAVES / 2; w++) x += *reinterpret_cast<const attn_f4*>(meet + (w * met_rows + r) * kStride + d);
    if (once) {
#pragma unroll
      for (int w = WAVES / 2; w < WAVES; w++) x += *reinterpret_cast<const attn_f4*>(meet + (w * met_rows + r) * kStride + d);
    }
    if (it.part < 0) {
      const AttnRow row = attn_row(a, it, kRows, r);
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = sum == 0.f ? (T)0.f : (T)(x[j] / sum);
      *reinterpret_cast<t4*>(static_cast<T*>(a.out) + ((long)(it.q_start + row.token) * (a.kv_heads * a.group) + head * a.group + row.head) * D + d) = y;
    } else {
      const long at = ((long)it.part * a.kv_heads + head) * (LIST == 2 ? kAttnPrefixRows : kRows) + r;
      *reinterpret_cast<attn_f4*>(a.part_o[LIST] + at * D + d) = x;
      if (d == 0) a.part_ml[LIST][2 * at] = top, a.part_ml[LIST][2 * at + 1] = sum;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Many rows: prompts.  Bound by the matrix cores and the exponentials.  A workgroup takes 128 rows, 32 a wavefront (as columns of 32 x 32 x 16
// MFMAs), and walks the share's tokens in blocks of 64 that all of it reads from LDS: two places, the next block on its way in registers,
// one barrier a block.  Codes of 8 bits become values on their way to LDS.  Two such workgroups a CU, so that one's exponentials run under the other's
// MFMAs, which have priority; K rows, and V rows for the transposing reads, are XOR-swizzled by 16-byte pieces (no bank conflicts).
// Measured: 4 x 500 new tokens in contexts of up to 8200, 64 heads over 8, bf16 338 us = 826 TFLOP/s (all four of 8200 910 - 940, in fp16 870 - 900); 4000 from the first on, 32
// heads, fp16 170 us = 771.  Counters of the first: matrix cores busy 41 % of the SIMDs' cycles, LDS 32 %, wavefronts waiting 29 % of theirs.  Loops of this MFMA reach
// 1660 TFLOP/s alone and 1330 with the softmax's 4 vector instructions and 2 exponentials each between them.  In e4m3, contexts of 8200, 780 - 810 in fp16 and 830 - 860 in bf16:
// conversions and scales.
// Measured and not kept: 256 rows on eight wavefronts and 128 tokens a barrier (equal contexts 1.02, e4m3 1.11, but 26 mixed sequences 0.87 and 3 x 100 new tokens
// 0.81), V of the first columns read ahead of the softmax (1.00), priority around the second product as well (1.00),
// the sums of P as one more product, of ones (0.99), three workgroups a CU for heads of 64 (16 bits 0.85; e4m3 1.06 on long batches, 0.8 to 0.9 on others).
template <int D>
struct AttnTileLds {
  static constexpr int kTile = kAttnBlock * 2 * D;
  alignas(16) uint8_t tiles[4 * kTile];                                                  // K, V, K, V
  alignas(16) float scales[2][2][kAttnBlock];
  int odd[2][4];                                                                         // infinities or NaNs among a wavefront's V
};

template <class T, int KIND, int D, bool GROUPS>
__device__ __forceinline__ void attend_tile(const AttendArgs& a, int index, int head, AttnTileLds<D>& shared) {
  using M = AttnMma<T>;
  using v8 = typename M::v8;
  constexpr int kRowBytes = 2 * D, kChunks = kRowBytes / 16, kKeyRows = 256 / kRowBytes;
  constexpr int kTile = AttnTileLds<D>::kTile;
  constexpr int kHeld = D * (KIND == kCacheSame ? 2 : 1), kHeldChunks = kHeld / 16;      // a row in the cache
  constexpr int kLoads = 16 * kHeldChunks / 64, kLoadRows = 64 / kHeldChunks;            // of the wavefront's 16 tokens of a block
  static_assert(kLoads >= 1, "16 tokens are a request at least");
  uint8_t* lds = shared.tiles;
  auto& scales = shared.scales;
  auto& odd = shared.odd;
  AttnItem it = attn_item(a, 1, index);
  if (index >= a.plan[2] || !attn_within(a, kAttnTileRows, &it)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;

  const int n_blocks = (it.kv_end - it.kv_begin + kAttnBlock - 1) / kAttnBlock;
  kv_uint4 rk[kLoads], rv[kLoads];
  float rs = 0.f;
  const int load_row = lane / kHeldChunks, load_chunk = lane % kHeldChunks;
  const int page_mask = (1 << a.page_shift) - 1;
  const AttnHeld<kLoadRows, false> held_k(a.ck, head, kHeld / D, load_row, load_chunk), held_v(a.cv, head, kHeld / D, load_row, load_chunk);
  const float *scale_k = a.ck.scale + head * a.ck.scale_head, *scale_v = a.cv.scale + head * a.cv.scale_head;
  // a lane fetches the page of the wavefront's 16 tokens of one of the next 64 blocks
  auto pages_from = [&](int i) {
    const long token = it.kv_begin + (long)(i + lane) * kAttnBlock + 16 * wave;
    return attn_page(a, it.seq, (int)min(token, (long)it.kv_end - 1));
  };
  int ids = n_blocks > 0 ? pages_from(0) : 0, next_ids = n_blocks > 64 ? pages_from(64) : 0;
  auto request = [&](int i) {
    if (i > 0 && i % 64 == 0) {
      ids = next_ids;
      if (n_blocks > i + 64) next_ids = pages_from(i + 64);
    }
    const long page = __builtin_amdgcn_readlane(ids, i % 64);
    const int slot = min(it.kv_begin + i * kAttnBlock + 16 * wave, (it.kv_end - 1) & ~15) & page_mask;
    held_k.template read<kLoads>(rk, page, slot);
    held_v.template read<kLoads>(rv, page, slot);
    if constexpr (KIND != kCacheSame)
      rs = lane < 16 ? scale_k[page * a.ck.scale_page + slot + lane] : scale_v[page * a.cv.scale_page + slot + (lane & 15)];
  };
  if (n_blocks > 0) request(0);
  const AttnRow mine = attn_row(a, it, kAttnTileRows, 32 * wave + col);
  const T* q = static_cast<const T*>(a.q) + attn_token<GROUPS>(a, it, mine.token) * a.q_token + (head * a.group + mine.head) * a.q_head;
  v8 qf[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; s++) qf[s] = mine.live ? *reinterpret_cast<const v8*>(q + 16 * s + 8 * h) : v8{0, 0, 0, 0, 0, 0, 0, 0};
  // the limits of the wavefront's and the tile's first and last rows: tokens between are the same for all of them
  const int n_rows = min(kAttnTileRows, it.n_tokens * a.group - it.tile * kAttnTileRows);
  const int wave_last = min(32 * wave + 31, n_rows - 1);
  const bool wave_live = 32 * wave < n_rows;
  const AttnRow w0 = attn_row(a, it, kAttnTileRows, 32 * wave), w1 = attn_row(a, it, kAttnTileRows, max(wave_last, 0));
  const AttnRow g0 = attn_row(a, it, kAttnTileRows, 0), g1 = attn_row(a, it, kAttnTileRows, n_rows - 1);

  auto key_of = [](int row) { return (row / kKeyRows) & (kChunks - 1); };
  auto key_of_v = [](int row) { return (row / kKeyRows << 2) & (kChunks - 1); };
  // the registers' 16 tokens of the block at t0 into place `at`
  auto keep = [&](int t0, int at) {
    uint8_t* to_k = lds + at * 2 * kTile;
    uint8_t* to_v = to_k + kTile;
    if (t0 + kAttnBlock > it.kv_end) {       // tokens behind the last: whatever the page holds there must not meet a zero of P
#pragma unroll
      for (int j = 0; j < kLoads; j++)
        if (t0 + 16 * wave + j * kLoadRows + load_row >= it.kv_end) rv[j] = kv_uint4{0, 0, 0, 0};
    }
    bool strange = false;
    if (t0 < g1.lo || t0 + kAttnBlock > g0.hi) {
#pragma unroll
      for (int j = 0; j < kLoads; j++) strange |= attn_clean<T, KIND>(&rv[j]);
    }
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int row = 16 * wave + j * kLoadRows + load_row;
      if constexpr (KIND == kCacheSame) {
        *reinterpret_cast<kv_uint4*>(to_k + row * kRowBytes + (load_chunk ^ key_of(row)) * 16) = rk[j];
        *reinterpret_cast<kv_uint4*>(to_v + row * kRowBytes + (load_chunk ^ key_of_v(row)) * 16) = rv[j];
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int chunk = 2 * load_chunk + i;
          *reinterpret_cast<v8*>(to_k + row * kRowBytes + (chunk ^ key_of(row)) * 16) = attn_values<T, KIND>(kv_uint2{rk[j][2 * i], rk[j][2 * i + 1]});
          *reinterpret_cast<v8*>(to_v + row * kRowBytes + (chunk ^ key_of_v(row)) * 16) = attn_values<T, KIND>(kv_uint2{rv[j][2 * i], rv[j][2 * i + 1]});
        }
      }
    }
    const bool any = __any(strange);
    if (lane == 0) odd[at][wave] = any;
    if constexpr (KIND != kCacheSame) {
      if (lane < 32) scales[at][lane / 16][16 * wave + (lane & 15)] = lane < 16 ? rs * a.scale_log2 : rs;
    }
  };

  // where a lane's K operand (row `col`, 16-byte piece h) and V operand (row 4 h + lane % 16 / 4, columns 16 (lane / 16 % 2) + 4 (lane % 4) ..) lie: piece 2 i
  // + h of K and 4 d + .. of V are an exclusive or away, other rows an offset, since the keys repeat every 16 rows (of V every 4)
  const int v_row = 4 * h + (lane & 15) / 4;
  const uint32_t lane_k = col * kRowBytes + (h ^ key_of(col)) * 16;
  const uint32_t lane_v = v_row * kRowBytes + ((2 * (lane >> 4 & 1) + (lane & 3) / 2) ^ key_of_v(v_row)) * 16 + 8 * (lane & 1);

  attn_f16 o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int j = 0; j < 16; j++) o[d][j] = 0.f;
  constexpr bool kNormed = KIND != kCacheSame && __is_same(T, _Float16);
  float m = kAttnNone, l = 0.f, peak = 0.f;  // l, o and peak are times 2^shift
  int shift = 0;

  if (n_blocks > 0) {
    keep(it.kv_begin, 0);
    if (n_blocks > 1) request(1);
  }
  __syncthreads();
  for (int block = 0; block < n_blocks; block++) {
    const int t0 = it.kv_begin + block * kAttnBlock, at = block & 1;
    auto step = [&] {                        // the next block into LDS, the one behind it requested
      if (block + 1 < n_blocks) {
        keep(t0 + kAttnBlock, at ^ 1);
        if (block + 2 < n_blocks) request(block + 2);
      }
    };
    if (!wave_live || t0 >= min(w1.hi, it.kv_end) || t0 + kAttnBlock <= w0.lo) {
      step();
    } else {
      // (one lane constant each, kept from being spread over a register for every address)
      uint32_t at_k = at * 2 * kTile + lane_k, at_v = at * 2 * kTile + kTile + lane_v;
      asm volatile("" : "+v"(at_k), "+v"(at_v));
      attn_f16 s[2];
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int j = 0; j < 16; j++) s[g][j] = 0.f;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int g = 0; g < 2; g++) s[g] = M::m32(*reinterpret_cast<const v8*>(lds + (at_k ^ (32 * i)) + 32 * g * kRowBytes), qf[i], s[g]);
      __builtin_amdgcn_s_setprio(0);
      step();                                // (its writes under the softmax)
      const bool edge = t0 < w1.lo || t0 + kAttnBlock > min(w0.hi, it.kv_end);
      const AttnSpan span = {mine.lo - t0 - 4 * h, min(mine.hi, it.kv_end) - t0 - 4 * h};
      float top = -__builtin_inff();
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
          if constexpr (KIND != kCacheSame) s[g][j] *= scales[at][0][32 * g + 8 * (j / 4) + j % 4 + 4 * h];
          top = fmaxf(top, s[g][j]);
        }
      if (edge) {
        const AttnSpan seen = span.here();
        top = -__builtin_inff();
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const int token = 32 * g + 8 * (j / 4) + j % 4;
            s[g][j] = seen.hides(token) ? -__builtin_inff() : s[g][j];
            top = fmaxf(top, s[g][j]);
          }
      }
      if constexpr (KIND == kCacheSame) top *= a.scale_log2;
      top = fmaxf(top, kAttnNone);
      top = attn_max32(top);
      if (__any(top > m + M::kHigh)) {
        const float low = top - M::kLow, next = fmaxf(m, kNormed ? __builtin_floorf(low) : low), f = __builtin_amdgcn_exp2f(m - next);
        l *= f, peak *= f, m = next;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
          for (int j = 0; j < 16; j++) o[d][j] *= f;
      }
      float under = kNormed ? m - (float)shift : m, to_log2 = KIND == kCacheSame ? a.scale_log2 : 1.f;
      if constexpr (KIND == kCacheSame || kNormed) {
        const bool far = attn_far(m);
        if (__any(far)) {
#pragma unroll
          for (int g = 0; g < 2; g++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[g][j] = KIND == kCacheSame ? s[g][j] * (far ? to_log2 : 1.f) : s[g][j] - (far ? m : 0.f);
          if (KIND == kCacheSame) to_log2 = far ? 1.f : to_log2;
          else under = far ? -(float)shift : under;
        }
      }
      v8 p[4];
      float sum[4] = {0.f, 0.f, 0.f, 0.f};   // (one running sum would be a chain of 32 additions)
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const float e = __builtin_amdgcn_exp2f(KIND == kCacheSame ? __builtin_fmaf(s[g][j], to_log2, -m) : s[g][j] - under);
          sum[j % 4] += e;
          s[g][j] = KIND == kCacheSame ? e : e * scales[at][1][32 * g + 8 * (j / 4) + j % 4 + 4 * h];
        }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (KIND != kCacheSame && edge) {              // (a scale may be a NaN)
        const AttnSpan seen = span.here();
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const int token = 32 * g + 8 * (j / 4) + j % 4;
            s[g][j] = seen.hides(token) ? 0.f : s[g][j];
          }
      }
      if constexpr (kNormed) {
        float most = 0.f;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int j = 0; j < 16; j++) most = fmaxf(most, __builtin_fabsf(s[g][j]));
        peak = fmaxf(peak, attn_max32(most));
        if (__any(attn_off(peak))) {
          const int by = attn_shift(peak, shift);
          shift += by, peak = __builtin_ldexpf(peak, by), l = __builtin_ldexpf(l, by);
#pragma unroll
          for (int g = 0; g < 2; g++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[g][j] = __builtin_ldexpf(s[g][j], by);
#pragma unroll
          for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[d][j] = __builtin_ldexpf(o[d][j], by);
        }
      }
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int j = 0; j < 16; j++) p[2 * g + j / 8][j % 8] = (T)s[g][j];
      auto column = [&](int d, int b) {      // V of 16 tokens from 16 b on, columns 32 d ..
        return attn_transposed<T>(lds, (at_v ^ (64 * d)) + 16 * b * kRowBytes, (at_v ^ (64 * d)) + (16 * b + 8) * kRowBytes);
      };
#pragma unroll
      for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int b = 0; b < 4; b++) o[d] = M::m32(column(d, b), p[b], o[d]);
      if ((t0 < g1.lo || t0 + kAttnBlock > g0.hi) && (odd[at][0] | odd[at][1] | odd[at][2] | odd[at][3])) {
#pragma unroll 1
        for (int token = t0; token < min(t0 + kAttnBlock, it.kv_end); token++) {
          const long page = attn_page(a, it.seq, token);
          const bool sees = token >= mine.lo && token < mine.hi;
#pragma unroll
          for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const attn_f4 x = attn_strange<T, KIND>(a.cv, page, head, token & ((1 << a.page_shift) - 1), 32 * d + 8 * i + 4 * h);
#pragma unroll
              for (int j = 0; j < 4; j++) o[d][4 * i + j] += sees ? x[j] : 0.f;
            }
        }
      }
    }
    __syncthreads();
  }
  if (!mine.live || 32 * wave + col >= n_rows) return;
  l += __shfl_xor(l, 32);
  float f = kNormed ? __builtin_ldexpf(1.f, -shift) : 1.f;
  if (it.part < 0) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    f = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(a.out) + ((long)(it.q_start + mine.token) * (a.kv_heads * a.group) + head * a.group + mine.head) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        t4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (T)(o[d][4 * i + j] * f);
        *reinterpret_cast<t4*>(out + 32 * d + 8 * i) = y;
      }
  } else {
    const long at = ((long)it.part * a.kv_heads + head) * kAttnTileRows + 32 * wave + col;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        attn_f4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = o[d][4 * i + j] * f;
        *reinterpret_cast<attn_f4*>(a.part_o[1] + at * D + 32 * d + 8 * i + 4 * h) = y;
      }
    if (h == 0) a.part_ml[1][2 * at] = m, a.part_ml[1][2 * at + 1] = l * f;
  }
}

// A batch of short sequences: a workgroup for every item and head of the cache.  grid list[0].max_items * kv_heads, block 64 WAVES
template <class T, int KIND, int D, int NQ, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void attend_rows_kernel(AttendArgs a) {
  __shared__ AttnRowsLds<KIND, D, NQ, WAVES> shared;
  const int index = blockIdx.x / a.kv_heads;
  attend_rows<T, KIND, D, NQ, WAVES>(a, index, blockIdx.x - index * a.kv_heads, shared);
}

// Any batch: the long list's items first, then the short one's, in one launch, so that what waits for memory runs beside what computes (a step of 26
// sequences, two of them of 203 and 177 new tokens, in e4m3: 36.9 and 19.5 us one after the other, 39.2 together).
// grid (list[1].max_items + list[0].max_items) * kv_heads, block 256
template <class T, int KIND, int D>
__global__ __launch_bounds__(256, 2) void attend_mixed_kernel(AttendArgs a) {
  __shared__ union {
    AttnTileLds<D> tile;
    AttnRowsLds<KIND, D, 1, 4> rows;
  } shared;
  const int index = blockIdx.x / a.kv_heads, head = blockIdx.x - index * a.kv_heads;
  if (index < a.list[1].max_items) attend_tile<T, KIND, D, false>(a, index, head, shared.tile);
  else attend_rows<T, KIND, D, 1, 4>(a, index - a.list[1].max_items, head, shared.rows);
}

// Batches in groups: long walks of few rows (prefixes, and sequences that share little), tiles of 128 rows (prefixes of many, prompts), then the sequences' own parts.
// SOLO: many of these, of few rows: a wavefront takes one and a head by itself, four of them a workgroup, and there is nothing to join between wavefronts.  (Of 220 tokens of a sequence's own a workgroup's
// four wavefronts walk two sub-tiles each and spend the rest of their time on the way there and on joining.)
// grid (list[2].max_items + list[1].max_items) * kv_heads + list[0].max_items * kv_heads (SOLO: a quarter of that, rounded up), block 256
template <class T, int KIND, int D, bool SOLO>
__global__ __launch_bounds__(256, 2) void attend_groups_kernel(AttendArgs a) {
  __shared__ union {
    AttnTileLds<D> tile;
    AttnRowsLds<KIND, D, 2, 4> prefix;
    AttnRowsLds<KIND, D, 1, 4> rows;
    AttnRowsLds<KIND, D, 1, 1> solo[4];
  } shared;
  const int prefixes = a.list[2].max_items, tiles = prefixes + a.list[1].max_items, index = blockIdx.x / a.kv_heads, head = blockIdx.x - index * a.kv_heads;
  if (index < prefixes) {
    const int* p = a.plan + a.list[2].items + 8L * index;        // (one tile each; behind the last item it does not matter)
    if (p[2] * a.group <= 16) attend_rows<T, KIND, D, 1, 4, 2>(a, index, head, shared.rows);
    else attend_rows<T, KIND, D, 2, 4, 2>(a, index, head, shared.prefix);
  } else if (index < tiles) {
    attend_tile<T, KIND, D, true>(a, index - prefixes, head, shared.tile);
  } else if constexpr (SOLO) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), unit = 4 * (blockIdx.x - tiles * a.kv_heads) + wave, own = unit / a.kv_heads;
    if (own < a.list[0].max_items) attend_rows<T, KIND, D, 1, 1>(a, own, unit - own * a.kv_heads, shared.solo[wave]);
  } else {
    attend_rows<T, KIND, D, 1, 4>(a, index - tiles, head, shared.rows);
  }
}

// Shares of one tile.  D / 4 lanes hold a row; a workgroup takes as many rows as it has such groups (or as many as there are, rounded up to a power of two) and,
// between them, the shares: a group adds every n-th share, the groups' sums are added in their order.  The host knows bounds only, mostly far above
// what there is to join, so a fixed number of workgroups walks what the plan says: one for every place of the bound took 10 to 15 us of a prompt's 180 to
// 370 to find that nothing was cut.  grid up to kAttnJoiners, block 256
constexpr int kAttnJoiners = 1024;
template <class T, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ attn_f4 sums[256];
  __shared__ float totals[kGroups];
  const int short_units = a.plan[1] * a.kv_heads * (a.list[0].rows / kGroups), units = short_units + a.plan[3] * a.kv_heads * (a.list[1].rows / kGroups);
  const int group = threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  for (int next = blockIdx.x; next < units; next += gridDim.x) {
    const int which = next < short_units ? 0 : 1, unit = next - (which ? short_units : 0);
    const int rows = a.list[which].rows, pieces = rows / kGroups, piece = unit % pieces, index = unit / pieces / a.kv_heads, head = unit / pieces - index * a.kv_heads;
    const int* j = a.plan + a.list[which].joins + 8L * index;
    const int q_start = j[0], n_tokens = j[1], tile = j[2], first = j[3], n_parts = j[4];
    const int r0 = kGroups * piece, live = min(kGroups, n_tokens * a.group - tile * rows - r0);
    if (live <= 0) continue;
    const float *part_o = a.part_o[which], *part_ml = a.part_ml[which];
    int wide = 1;                                  // rows side by side
    while (wide < live) wide *= 2;
    const int i = group % wide, n = kGroups / wide;
    const long step = (long)a.kv_heads * rows, at = ((long)first * a.kv_heads + head) * rows + r0 + min(i, live - 1);
    float top = kAttnNone, sum = 0.f;
#pragma unroll 4
    for (int p = 0; p < n_parts; p++) top = fmaxf(top, part_ml[2 * (at + p * step)]);
    attn_f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = group / wide; p < n_parts; p += n) {
      const float f = __builtin_amdgcn_exp2f(part_ml[2 * (at + p * step)] - top);
      sum += f * part_ml[2 * (at + p * step) + 1];
      const attn_f4 y = *reinterpret_cast<const attn_f4*>(part_o + (at + p * step) * D + d);
#pragma unroll
      for (int k = 0; k < 4; k++) x[k] = __builtin_fmaf(y[k], f, x[k]);
    }
    sums[threadIdx.x] = x;
    if (d == 0) totals[group] = sum;
    __syncthreads();
    if (group < live) {
      for (int g = 1; g < n; g++) {
        x += sums[threadIdx.x + g * wide * kLanes];
        sum += totals[group + g * wide];
      }
      const int row = tile * rows + r0 + group, token = row / a.group, g = row - token * a.group;
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
#pragma unroll
      for (int k = 0; k < 4; k++) y[k] = sum == 0.f ? (T)0.f : (T)(x[k] / sum);
      *reinterpret_cast<t4*>(static_cast<T*>(a.out) + ((long)(q_start + token) * (a.kv_heads * a.group) + head * a.group + g) * D + d) = y;
    }
    __syncthreads();
  }
}

// The same for batches in groups that share a prefix: a tile of a group has the shares of its group's prefix behind its own, in the prefix's tiles that hold its rows.  Every
// row is joined, so this is as long as its round trips: a lane group requests eight shares at once, statistics and sums together, and takes them in under a
// running maximum; the plan says how many rows the fullest tile has, so that a unit has work.  Two passes over the shares, one for the maxima, over all
// places of the tiles took 14 us for 64 requests of 64 heads and 23 for 96 of 32 + 32, this 7 and 11.  grid up to kAttnJoiners, block 256
template <class T, int D>
__global__ __launch_bounds__(256) void attend_join_shared_kernel(AttendArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes, kAtOnce = 8;
  __shared__ attn_f4 sums[256];
  __shared__ float tops[kGroups], totals[kGroups];
  int pieces[kAttnLists], units[kAttnLists];
#pragma unroll
  for (int which = 0; which < kAttnLists; which++) {
    pieces[which] = (a.plan[6 + which] + kGroups - 1) / kGroups;
    units[which] = a.plan[2 * which + 1] * a.kv_heads * pieces[which];
  }
  const int group = threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  for (int next = blockIdx.x; next < units[0] + units[1] + units[2]; next += gridDim.x) {
    const int which = next < units[0] ? 0 : next < units[0] + units[1] ? 1 : 2, unit = next - (which > 0 ? units[0] : 0) - (which > 1 ? units[1] : 0);
    const int per = which == 0 ? pieces[0] : which == 1 ? pieces[1] : pieces[2];
    const int rows = a.list[which].rows, piece = unit % per, index = unit / per / a.kv_heads, head = unit / per - index * a.kv_heads;
    const int* j = a.plan + a.list[which].joins + 8L * index;
    const int q_start = j[0], n_tokens = j[1], tile = j[2], first = j[3], n_own = j[4], prefix_list = j[5], prefix_tile = j[6], prefix_row = j[7];
    const int r0 = kGroups * piece, live = min(min(kGroups, rows - r0), n_tokens * a.group - tile * rows - r0);
    if (live <= 0) continue;
    int wide = 1;                                  // rows side by side
    while (wide < live) wide *= 2;
    const int i = group % wide, n = kGroups / wide, mine = r0 + min(i, live - 1);
    const long step = (long)a.kv_heads * rows, at = ((long)first * a.kv_heads + head) * rows + mine;
    const float *own_o = a.part_o[which], *own_ml = a.part_ml[which], *prefix_o = own_o, *prefix_ml = own_ml;
    int n_parts = n_own;
    long prefix_step = 0, prefix_at = 0;
    if (prefix_list >= 0) {
      const int prefix_rows = a.list[prefix_list].rows, row = prefix_row + tile * rows + mine;
      const int* p = a.plan + a.list[prefix_list].prefixes + 2L * (prefix_tile + row / prefix_rows);
      prefix_o = a.part_o[prefix_list], prefix_ml = a.part_ml[prefix_list], prefix_step = (long)a.kv_heads * prefix_rows;
      prefix_at = ((long)p[0] * a.kv_heads + head) * prefix_rows + row % prefix_rows, n_parts += p[1];
    }
    float top = kAttnNone, sum = 0.f;
    attn_f4 x = {0.f, 0.f, 0.f, 0.f};
    typedef float ml2 __attribute__((ext_vector_type(2)));
    for (int p0 = group / wide; p0 < n_parts; p0 += kAtOnce * n) {
      ml2 ml[kAtOnce];
      attn_f4 o[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const int p = p0 + k * n;
        const bool own = p < n_own;
        const long place = own ? at + p * step : prefix_at + (p - n_own) * prefix_step;
        ml[k] = ml2{kAttnNone, 0.f}, o[k] = attn_f4{0.f, 0.f, 0.f, 0.f};
        if (p < n_parts) ml[k] = reinterpret_cast<const ml2*>(own ? own_ml : prefix_ml)[place], o[k] = *reinterpret_cast<const attn_f4*>((own ? own_o : prefix_o) + place * D + d);
      }
      float high = top;
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) high = fmaxf(high, ml[k].x);
      const float back = __builtin_amdgcn_exp2f(top - high);
      sum *= back, x *= back, top = high;
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const float f = p0 + k * n < n_parts ? __builtin_amdgcn_exp2f(ml[k].x - top) : 0.f;
        sum = __builtin_fmaf(f, ml[k].y, sum);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(o[k][e], f, x[e]);
      }
    }
    if (n > 1) {
      sums[threadIdx.x] = x;
      if (d == 0) tops[group] = top, totals[group] = sum;
      __syncthreads();
      if (group < live) {
        float high = top;
        for (int g = 1; g < n; g++) high = fmaxf(high, tops[group + g * wide]);
        float f = __builtin_amdgcn_exp2f(top - high);
        sum *= f, x *= f;
        for (int g = 1; g < n; g++) {
          f = __builtin_amdgcn_exp2f(tops[group + g * wide] - high);
          sum = __builtin_fmaf(f, totals[group + g * wide], sum);
          x += sums[threadIdx.x + g * wide * kLanes] * f;
        }
      }
    }
    if (group < live) {
      const int row = tile * rows + r0 + group, token = row / a.group, g = row - token * a.group;
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
#pragma unroll
      for (int k = 0; k < 4; k++) y[k] = sum == 0.f ? (T)0.f : (T)(x[k] / sum);
      *reinterpret_cast<t4*>(static_cast<T*>(a.out) + ((long)(q_start + token) * (a.kv_heads * a.group) + head * a.group + g) * D + d) = y;
    }
    __syncthreads();
  }
}

}  // namespace triteia_hip
