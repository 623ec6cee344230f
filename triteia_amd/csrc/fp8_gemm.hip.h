// y[t, j] = sum over blocks b of 128 k of  x_scale[t, b] w_scale[j / 128, b] sum_{i in b} x[t, i] w[j, i]
//
// x [tokens, k] and w [m, k] in e4m3, rows of adjacent codes.  A block is one 16 x 16 x 128 MFMA: its sums start at zero and go into the running 32-bit sums by one
// fma with the product of both scales, which a lane has to know for its token only (weights are the MFMA's rows, tokens its columns; a wavefront's features lie
// in one block of 128).
//
// What the instruction does inside a block, measured: it adds the products of eight adjacent codes in fixed point, down to 2^-13 of the largest of the eight,
// and these sums in 32 bits.  Random codes come out 1.3e-5 off in norm; the codes themselves are 2e-2 off what they stand for.  Sums that are exact to 32 bits would take the
// instruction of 16 bits on widened codes, at half the rate.
#pragma once
#include "fp8_quant.hip.h"
#include "sparse24_gemm.hip.h"

namespace triteia_hip {

struct Fp8Args {
  const uint8_t* x;       // [tokens, k] (fp8_stream_kernel on 16 bits: of those)
  long x_stride;          // up to 2^24, as w_stride: a tile's rows are 32-bit offsets apart
  const float* xs;        // [tokens, blocks] by strides
  long xs_token, xs_block;
  const uint8_t* w;       // [m, k]
  long w_stride;
  const float* ws;        // [m / 128, blocks]
  long ws_row, ws_block;
  void* out;              // [tokens, m]
  int type;               // of out: 0 fp16, 1 bf16, 2 fp32
  int tokens, m, k;       // k a multiple of 16
  int splits;             // shares of K over workgroups; 1: the result goes to `out`
  int rotate;             // 1: feature groups start their walks over K spread around its blocks, 0: at the first
  float* partial;         // [splits][tokens][m] (splits > 1)
};

constexpr int kFp8Band = 4;

typedef int fp8_v8 __attribute__((ext_vector_type(8)));

// 4 bytes a lane to `lds` (uniform) + 4 lane; the caller waits (see direct_load)
__device__ __forceinline__ void direct_load4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "{m0}"(lds) : "memory");
}

__device__ __forceinline__ float4_t fp8_mma(const fp8_v8& a, const fp8_v8& b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ fp8_v8 fp8_operand(const unsigned char* row, int piece) {      // pieces of 16 codes, and the one 64 further on
  union { fp8_v8 v; uint4_t h[2]; } u;
  u.h[0] = *reinterpret_cast<const uint4_t*>(row + piece);
  u.h[1] = *reinterpret_cast<const uint4_t*>(row + (piece ^ 64));
  return u.v;
}

// four results of a row of m, from the j0-th on
template <class T>
__device__ __forceinline__ void fp8_store(T* to, const float4_t& v, int m, int j0) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  if (m % 4 == 0) {
    *reinterpret_cast<t4*>(to) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else {
    for (int j = 0; j < 4; j++)
      if (j0 + j < m) to[j] = (T)v[j];
  }
}

__device__ __forceinline__ void fp8_result(const Fp8Args& p, int share, int token, int j0, const float4_t& v) {
  const long at = (long)token * p.m + j0;
  if (p.splits > 1) fp8_store<float>(p.partial + (long)share * p.tokens * p.m + at, v, p.m, j0);
  else if (p.type == 0) fp8_store<_Float16>(static_cast<_Float16*>(p.out) + at, v, p.m, j0);
  else if (p.type == 1) fp8_store<__bf16>(static_cast<__bf16*>(p.out) + at, v, p.m, j0);
  else fp8_store<float>(static_cast<float*>(p.out) + at, v, p.m, j0);
}

// NT x F: 16-token by 16-feature tiles of a wavefront; TW x FW wavefronts side by side.  Both operands go through LDS by direct loads, a ring of STAGES blocks.
//
// Few tiles are bound by the weights' way from HBM: 64 tokens in codes on 8192 x 28672, four weights in turn, 48 us (4.9 TB/s; 56 before the walks were spread over K); the same weight
// again and again, which the Infinity Cache holds, 36 either way.  The large one, 256 x 256 on eight
// wavefronts, by the matrix cores and what stands between their instructions: 8000 tokens on 8192 x 28672 1600 to 1680 us, 2240 to 2350 TFLOP/s; 1520 without the additions
// (every second slot of the vector ALUs), 1350 without loads, 1180 without both.  Counted there: matrix cores busy 60 % of the cycles, at 1.9 GHz; LDS 27 %, no conflicts; wavefronts
// wait 27 % of theirs; 2.8 GB read beyond L2, 0.3 of them once, at 1.7 TB/s.  (A library product with one scale a tensor, which has no additions, takes 1286.)
// Measured and left: four wavefronts of 96 x 128 or 64 x 128, which read less of LDS (2246 and 2724 us: one wavefront a SIMD does not hide its own MFMAs), weights from L2 to
// registers past LDS (3650), 32 x 32 x 64 instructions (192 x 256 1960 -> 2200; 256 x 256 passes the registers), requests two blocks ahead, priorities.
template <int NT, int TW, int F, int FW, int STAGES>
struct Fp8Tile {
  static constexpr int kTokens = 16 * NT * TW, kFeatures = 16 * F * FW;
  static constexpr int kWaves = TW * FW, kThreads = 64 * kWaves;
  static constexpr int kCodes = 128 * (kTokens + kFeatures), kScales = 256 * kWaves;
  static constexpr int kStageBytes = kCodes + kScales;
  static constexpr int kWeightScales = (kFeatures + 127) / 128;
  static constexpr int kLdsBytes = STAGES * kStageBytes;
  static_assert(16 * F <= 128 && 128 % (16 * F) == 0 && kTokens + kWeightScales <= 64 * kWaves && kFeatures % 8 == 0, "");
};

// all but the newest MOST sets of requests, or as many as there are behind the block
template <int MOST, int LOADS>
__device__ __forceinline__ void fp8_wait(int behind) {
  if constexpr (MOST > 0) {
    if (behind < MOST) return fp8_wait<MOST - 1, LOADS>(behind);
  }
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(MOST * LOADS) : "memory");
}

template <int NT, int TW, int F, int FW, int STAGES>
__global__ __launch_bounds__(64 * TW * FW) void fp8_tile_kernel(const Fp8Args p) {
  using Tile = Fp8Tile<NT, TW, F, FW, STAGES>;
  constexpr int TT = Tile::kTokens, FF = Tile::kFeatures, WAVES = Tile::kWaves;
  constexpr int kXLoads = (TT / 8 + WAVES - 1) / WAVES, kWLoads = (FF / 8 + WAVES - 1) / WAVES;
  constexpr int kLoads = kXLoads + kWLoads + 1;      // a wavefront's requests per block: the same in all of them (a few are made twice)
  constexpr int AHEAD = STAGES - 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int tw = wave / FW, fw = wave % FW;

  // Units: token tiles in bands of kBand, in a band (feature group, share of K, token tile), token tiles fastest.  An XCD (workgroup u runs on XCD u % 8) takes a run of
  // them, so that what runs there at once is a band's token tiles on a few feature groups and its L2 serves both.
  const int ttiles = (p.tokens + TT - 1) / TT, groups = (p.m + FF - 1) / FF;
  const int units = ttiles * groups * p.splits;
  const int per_xcd = (units + 7) >> 3;
  const int u = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || u >= units) return;
  const int band = u / (kFp8Band * groups * p.splits), in_band = u - band * (kFp8Band * groups * p.splits), deep = min(kFp8Band, ttiles - kFp8Band * band);
  const int tt = kFp8Band * band + in_band % deep, z = (in_band / deep) % p.splits, fg = in_band / (deep * p.splits);
  const int t0 = tt * TT, f0 = fg * FF;
  const int blocks = (p.k + 127) >> 7;
  const int c0 = (int)((long)z * blocks / p.splits), n = (int)((long)(z + 1) * blocks / p.splits) - c0;
  const int rot = p.rotate ? (int)((long)fg * n / groups) : 0;

  // A request: 8 rows x 128 bytes; lane l takes 16 bytes of row l / 8, the piece (l % 8) ^ (l / 8) to position l % 8.
  // (rows past the end repeat the last one: their sums are not stored; a tile's rows lie within 2^32 bytes)
  const uint8_t *x0 = p.x + (long)t0 * p.x_stride + 128L * c0, *w0 = p.w + (long)f0 * p.w_stride + 128L * c0;
  uint32_t src[kLoads - 1], dst[kLoads - 1];
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  const int lane_piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < kLoads - 1; i++) {
    const bool is_x = i < kXLoads;
    const int g = min(wave + WAVES * (is_x ? i : i - kXLoads), (is_x ? TT : FF) / 8 - 1), row = 8 * g + (lane >> 3);
    src[i] = (is_x ? (uint32_t)min(row, p.tokens - 1 - t0) * (uint32_t)p.x_stride : (uint32_t)min(row, p.m - 1 - f0) * (uint32_t)p.w_stride) + 16 * lane_piece;
    dst[i] = lds0 + (is_x ? 0 : 128 * TT) + 1024 * g;
  }
  // scales of a block: those of the tile's tokens, then those of its weights' blocks, 64 a wavefront
  const int which = 64 * wave + lane;
  const float* scale_src = which < TT ? p.xs + (long)min(t0 + which, p.tokens - 1) * p.xs_token + c0 * p.xs_block
                                      : p.ws + (long)min((f0 >> 7) + min(which - TT, Tile::kWeightScales - 1), (p.m - 1) >> 7) * p.ws_row + c0 * p.ws_block;
  const long scale_step = which < TT ? p.xs_block : p.ws_block;
  // The last block of a K that ends inside it: lanes whose piece lies behind the end read the block's first piece instead, and put zeros in its place in LDS.
  const int odd_block = p.k % 128 ? blocks - 1 - c0 : -1;
  const uint32_t back = 128 * (blocks - 1) + 16 * lane_piece >= p.k ? 16 * lane_piece : 0;
  auto block_of = [&](int c) { return c + rot < n ? c + rot : c + rot - n; };      // the c-th of the walk
  auto issue = [&](int i, int c, int stage) {
    if (i == kLoads - 1) {
      direct_load4(scale_src + c * scale_step, __builtin_amdgcn_readfirstlane(lds0 + stage * Tile::kStageBytes + Tile::kCodes + 256 * wave));
    } else {
      const uint8_t* base = (i < kXLoads ? x0 : w0) + 128L * c;
      direct_load(src[i] - (c == odd_block ? back : 0), base, __builtin_amdgcn_readfirstlane(dst[i] + stage * Tile::kStageBytes));
    }
  };
  auto clear = [&](int stage) {
    if (back == 0) return;
#pragma unroll
    for (int i = 0; i < kLoads - 1; i++) *reinterpret_cast<uint4_t*>(smem + (dst[i] - lds0) + stage * Tile::kStageBytes + 16 * lane) = uint4_t{0, 0, 0, 0};
  };

  float4_t acc[F][NT], d[F];
#pragma unroll
  for (int f = 0; f < F; f++) {
    d[f] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; t++) acc[f][t] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  float scale = 0.f;                                       // of the sums in d
  const int piece = (q ^ (r & 7)) * 16;
  const uint32_t xrow = (16 * NT * tw + r) * 128;
  const uint32_t wrow = 128 * TT + (16 * F * fw + r) * 128;
  // A block: between the MFMAs of one token tile the sums of the tile before it are added, so that neither waits for the other; the last tile's are added
  // in the next block.
  auto add = [&](int f, int t) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc[f][t][j] = __builtin_fmaf(d[f][j], scale, acc[f][t][j]);
  };
  auto compute = [&](int stage, auto&& request) {
    const unsigned char* s = smem + stage * Tile::kStageBytes;
    const float* scales = reinterpret_cast<const float*>(s + Tile::kCodes);
    const float sw = scales[TT + 16 * F * fw / 128];
    fp8_v8 w[F], x = fp8_operand(s + xrow, piece);
    float next = scales[16 * NT * tw + r];
#pragma unroll
    for (int f = 0; f < F; f++) w[f] = fp8_operand(s + wrow + 2048 * f, piece);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const fp8_v8 now = x;
      const float mine = next * sw;
      if (t + 1 < NT) x = fp8_operand(s + xrow + 2048 * (t + 1), piece), next = scales[16 * (NT * tw + t + 1) + r];
#pragma unroll
      for (int f = 0; f < F; f++) {
        add(f, t == 0 ? NT - 1 : t - 1);
        d[f] = fp8_mma(w[f], now);
        __builtin_amdgcn_sched_barrier(0);
      }
      scale = mine;
      constexpr int kEach = 4 * NT < kLoads ? (kLoads + NT - 1) / NT : 4;      // (early: the last of them have the rest of the block to arrive)
#pragma unroll
      for (int i = t * kEach; i < (t + 1) * kEach && i < kLoads; i++) request(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  for (int c = 0; c < AHEAD && c < n; c++)
#pragma unroll
    for (int i = 0; i < kLoads; i++) issue(i, block_of(c), c);
  // AHEAD blocks are in flight at the top, kLoads requests each, and complete in order: all but the newest AHEAD - 1 sets done means that this wavefront's part
  // of block c has landed.  The barrier makes all parts visible and says that every wavefront has read the block before, whose stage takes block c + AHEAD.
  // (One loop with a branch around the requests would hold the sums twice.)
  int c = 0, stage = 0;
  for (; c + AHEAD < n; c++) {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"((AHEAD - 1) * kLoads) : "memory");
    if (block_of(c) == odd_block) clear(stage);
    lds_barrier();
    const int free_stage = stage == 0 ? STAGES - 1 : stage - 1, ahead = block_of(c + AHEAD);
    compute(stage, [&](int i) { issue(i, ahead, free_stage); });
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  for (; c < n; c++) {
    fp8_wait<AHEAD - 1, kLoads>(n - 1 - c);
    if (block_of(c) == odd_block) clear(stage);
    lds_barrier();
    compute(stage, [](int) {});
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
#pragma unroll
  for (int f = 0; f < F; f++) add(f, NT - 1);

  // D: lane (token r, q) holds features 4q .. 4q + 3 of a tile
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int token = t0 + 16 * (NT * tw + t) + r;
#pragma unroll
    for (int f = 0; f < F; f++) {
      const int j0 = f0 + 16 * (F * fw + f) + 4 * q;
      if (token < p.tokens && j0 < p.m) fp8_result(p, z, token, j0, acc[f][t]);
    }
  }
}

// Few tokens: bound by the weights' way from HBM, on small layers by a launch and its round trips.  A workgroup takes 16 F features and 16 NT tokens at most; its
// wavefronts take turns at the blocks of K, each with a ring of its own in LDS, so that nothing is waited for but a wavefront's own requests; their sums
// meet once at the end.
// T: what x holds, codes (uint8_t) or, for up to 4 tokens, values of 16 bits that the wavefront quantises block by block (as fp8_quant_rows_kernel does, 16 lanes a
// row), every workgroup for itself: a launch less, and no scratch.
template <class T, int NT, int F, int WAVES, int STAGES>
struct Fp8Stream {
  static constexpr bool kQuant = !__is_same(T, uint8_t);
  static constexpr int kTokens = 16 * NT, kFeatures = 16 * F, kThreads = 64 * WAVES;
  static constexpr int kXLoads = kQuant ? 1 : kTokens / 8, kWLoads = kFeatures / 8;
  static constexpr int kScaleLoads = kQuant ? 1 : (kTokens + 1 + 63) / 64;
  static constexpr int kCodes = 1024 * (kXLoads + kWLoads), kStageBytes = kCodes + 256 * kScaleLoads;
  static constexpr int kOwnBytes = kQuant ? 128 * kTokens + 4 * kTokens : 0;       // a wavefront's codes and scales of the block that it multiplies
  static constexpr int kWaveBytes = STAGES * kStageBytes + kOwnBytes;
  static constexpr int kMeet = WAVES * kTokens * (kFeatures + 4) * 4;
  static constexpr int kLdsBytes = WAVES * kWaveBytes > kMeet ? WAVES * kWaveBytes : kMeet;
  static_assert(!kQuant || (NT == 1 && kOwnBytes % 16 == 0), "");
};

template <class T, int NT, int F, int WAVES, int STAGES>
__global__ __launch_bounds__(64 * WAVES) void fp8_stream_kernel(const Fp8Args p) {
  using Tile = Fp8Stream<T, NT, F, WAVES, STAGES>;
  constexpr int TT = Tile::kTokens, FF = Tile::kFeatures, kXLoads = Tile::kXLoads, kWLoads = Tile::kWLoads, kLoads = kXLoads + kWLoads + Tile::kScaleLoads, AHEAD = STAGES - 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int ttiles = (p.tokens + TT - 1) / TT, groups = (p.m + FF - 1) / FF, units = ttiles * groups * p.splits, per_xcd = (units + 7) >> 3;
  const int u = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || u >= units) return;
  const int tt = u % ttiles, z = (u / ttiles) % p.splits, fg = u / (ttiles * p.splits);
  const int t0 = tt * TT, f0 = fg * FF;
  const int blocks = (p.k + 127) >> 7;
  const int c0 = (int)((long)z * blocks / p.splits), all = (int)((long)(z + 1) * blocks / p.splits) - c0;
  const int rot = p.rotate ? (int)((long)fg * all / groups) : 0;
  const int n = wave < all ? (all - wave + WAVES - 1) / WAVES : 0;      // of the wavefront

  constexpr int kXBlock = Tile::kQuant ? 256 : 128;                     // bytes of a row
  const uint8_t *x0 = p.x + (long)t0 * p.x_stride * (kXBlock / 128) + (long)kXBlock * c0, *w0 = p.w + (long)f0 * p.w_stride + 128L * c0;
  uint32_t src[kXLoads + kWLoads];
  const int lane_piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < kXLoads + kWLoads; i++) {
    const bool is_x = i < kXLoads;
    const int row = 8 * (is_x ? i : i - kXLoads) + (lane >> 3);
    src[i] = (is_x ? (uint32_t)min(row, p.tokens - 1 - t0) * (uint32_t)p.x_stride : (uint32_t)min(row, p.m - 1 - f0) * (uint32_t)p.w_stride) + 16 * lane_piece;
    if (Tile::kQuant && is_x) src[i] = (uint32_t)min(q, p.tokens - 1) * (uint32_t)p.x_stride * 2 + 16 * r;      // 4 rows in a request
  }
  const float* scale_src[Tile::kScaleLoads];
  long scale_step[Tile::kScaleLoads];
#pragma unroll
  for (int i = 0; i < Tile::kScaleLoads; i++) {
    const int e = 64 * i + lane;
    const bool is_x = !Tile::kQuant && e < TT;
    scale_src[i] = is_x ? p.xs + (long)min(t0 + e, p.tokens - 1) * p.xs_token + c0 * p.xs_block : p.ws + (long)(f0 >> 7) * p.ws_row + c0 * p.ws_block;
    scale_step[i] = is_x ? p.xs_block : p.ws_block;
  }
  // (a last block that is not whole: as in fp8_tile_kernel)
  const int odd_block = p.k % 128 ? blocks - 1 - c0 : -1;
  const uint32_t back = 128 * (blocks - 1) + 16 * lane_piece >= p.k ? 16 * lane_piece : 0, back_x = 128 * (blocks - 1) + 8 * r >= p.k ? 16 * r : 0;
  const uint32_t ring = wave * Tile::kWaveBytes, lds0 = (uint32_t)(uintptr_t)smem + ring;
  auto block_of = [&](int c) {
    const int b = wave + WAVES * c + rot;
    return b < all ? b : b - all;
  };
  auto issue = [&](int c, int stage) {
    const int b = block_of(c);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + stage * Tile::kStageBytes), less = b == odd_block ? back : 0, less_x = b != odd_block ? 0 : Tile::kQuant ? back_x : back;
#pragma unroll
    for (int i = 0; i < kXLoads + kWLoads; i++) {
      if (i < kXLoads) direct_load(src[i] - less_x, x0 + (long)kXBlock * b, to + 1024 * i);
      else direct_load(src[i] - less, w0 + 128L * b, to + 1024 * i);
    }
#pragma unroll
    for (int i = 0; i < Tile::kScaleLoads; i++) direct_load4(scale_src[i] + b * scale_step[i], to + Tile::kCodes + 256 * i);
  };

  float4_t acc[F][NT];
#pragma unroll
  for (int f = 0; f < F; f++)
#pragma unroll
    for (int t = 0; t < NT; t++) acc[f][t] = float4_t{0.f, 0.f, 0.f, 0.f};
  const int piece = (q ^ (r & 7)) * 16;
  auto compute = [&](int c, int stage) {
    unsigned char* s = smem + ring + stage * Tile::kStageBytes;
    const bool odd = block_of(c) == odd_block;
    if (odd && back != 0) {
#pragma unroll
      for (int i = Tile::kQuant ? kXLoads : 0; i < kXLoads + kWLoads; i++) *reinterpret_cast<uint4_t*>(s + 1024 * i + 16 * lane) = uint4_t{0, 0, 0, 0};
    }
    const float* scales = reinterpret_cast<const float*>(s + Tile::kCodes);
    const float sw = scales[Tile::kQuant ? 0 : TT];
    unsigned char* own = Tile::kQuant ? smem + ring + STAGES * Tile::kStageBytes : s;
    float* own_scales = reinterpret_cast<float*>(Tile::kQuant ? own + 128 * TT : s + Tile::kCodes);
    if constexpr (Tile::kQuant) {
      kv8<T> v = *reinterpret_cast<const kv8<T>*>(s + 16 * lane);
      if (odd && back_x != 0) v = kv8<T>{0, 0, 0, 0, 0, 0, 0, 0};
      float scale;
      const kv_uint2 code = fp8_quantised<T>(v, &scale);
      *reinterpret_cast<kv_uint2*>(own + 128 * q + ((r / 2) ^ q) * 16 + 8 * (r & 1)) = code;
      if (r == 0) own_scales[q] = scale;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");      // (the wavefront's own: its lanes run together)
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }
    fp8_v8 w[F], x[NT];
    float scale[NT];
#pragma unroll
    for (int f = 0; f < F; f++) w[f] = fp8_operand(s + 1024 * kXLoads + 2048 * f + 128 * r, piece);
#pragma unroll
    for (int t = 0; t < NT; t++) x[t] = fp8_operand(own + 2048 * t + 128 * r, piece), scale[t] = own_scales[16 * t + r] * sw;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int f = 0; f < F; f++) {
        const float4_t d = fp8_mma(w[f], x[t]);
#pragma unroll
        for (int j = 0; j < 4; j++) acc[f][t][j] = __builtin_fmaf(d[j], scale[t], acc[f][t][j]);
      }
  };

#pragma unroll
  for (int c = 0; c < AHEAD; c++)
    if (c < n) issue(c, c);
  int stage = 0;
  for (int c = 0; c < n; c++) {
    // (the place that block c + AHEAD takes was read in the turn before)
    if (c + AHEAD < n) issue(c + AHEAD, stage == 0 ? STAGES - 1 : stage - 1);
    fp8_wait<AHEAD, kLoads>(n - 1 - c);
    compute(c, stage);
    __builtin_amdgcn_sched_barrier(0);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }

  // the wavefronts' sums, in their order
  __syncthreads();
  float* meet = reinterpret_cast<float*>(smem);
  constexpr int kStride = FF + 4;
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int f = 0; f < F; f++) *reinterpret_cast<float4_t*>(meet + (wave * TT + 16 * t + r) * kStride + 16 * f + 4 * q) = acc[f][t];
  __syncthreads();
  for (int e = threadIdx.x; e < TT * FF / 4; e += Tile::kThreads) {
    const int token = e / (FF / 4), j = 4 * (e % (FF / 4));
    if (t0 + token >= p.tokens || f0 + j >= p.m) continue;
    float4_t sum = *reinterpret_cast<const float4_t*>(meet + token * kStride + j);
#pragma unroll
    for (int w = 1; w < WAVES; w++) sum += *reinterpret_cast<const float4_t*>(meet + (w * TT + token) * kStride + j);
    fp8_result(p, z, t0 + token, f0 + j, sum);
  }
}

// The shares of K, added in order and rounded once; 4 results a thread (or one, where rows do not divide by 4).
template <class T, int N>
__global__ __launch_bounds__(256) void fp8_reduce_kernel(const float* __restrict__ partial, int splits, long results, T* __restrict__ out) {
  typedef float vN __attribute__((ext_vector_type(N)));
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * N;
  if (e >= results) return;
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; i++) sum[i] = 0.f;
#pragma unroll 4
  for (int z = 0; z < splits; z++) {
    const vN v = *reinterpret_cast<const vN*>(partial + z * results + e);
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] += v[i];
  }
#pragma unroll
  for (int i = 0; i < N; i++) out[e + i] = (T)sum[i];
}

}  // namespace triteia_hip
