// C entry points of the product in 8 bits and its quantiser (fp8_quant.hip.h, fp8_gemm.hip.h); part of triteia_hip.hip.
#pragma once

namespace {

constexpr int kFp8Most = 1 << 24;        // rows, columns and features of one call

int check_fp8(const char* what, int n, int k) {
  if (n < 0 || k < 0 || n > kFp8Most || k > kFp8Most || k % 16 != 0)
    return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d rows of %d elements: a multiple of 16, up to 2^24", what, n, k);
  return TRITEIA_HIP_OK;
}
int fp8_blocks(int k) { return (k + kFp8Block - 1) / kFp8Block; }

// 16 rows x U blocks a workgroup of the quantiser: one block while all of them fit side by side, four of a large tensor, requested together.  (us, one / four, on rows of 8192 in
// fp16, four tensors in turn and the same one again: 128 2.4 / 3.2 and 2.4 / 3.1, 512 4.4 / 4.8 and 3.9 / 4.1, 1024 7.2 / 7.3 and 5.9 / 5.8, 8000 41 / 37.5 and 33 / 32.)
long fp8_groups(int n, int k, int u) { return (n + 15L) / 16 * ((fp8_blocks(k) + u - 1) / u); }
constexpr int kFp8Wide = 4;
int fp8_width(int n, int k) { return fp8_groups(n, k, 1) > 2048 ? kFp8Wide : 1; }

template <class T>
int launch_fp8_quant(const Fp8QuantArgs& a, int rows, hipStream_t st) {
  if (rows != 1) {
    hipLaunchKernelGGL(fp8_quant_tiles_kernel<T>, dim3((unsigned)((a.n + 127L) / 128 * fp8_blocks(a.k))), dim3(256), 0, st, a);
    return check_launch("fp8_quant_tiles_kernel");
  }
  const int u = fp8_width(a.n, a.k);
  const dim3 grid((unsigned)fp8_groups(a.n, a.k, u));
  if (u == 1) hipLaunchKernelGGL((fp8_quant_rows_kernel<T, 1>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((fp8_quant_rows_kernel<T, kFp8Wide>), grid, dim3(256), 0, st, a);
  return check_launch("fp8_quant_rows_kernel");
}
template <class T>
void launch_fp8_values(const Fp8ValuesArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(fp8_values_kernel<T>, dim3((unsigned)fp8_groups(a.n, a.k, 1)), dim3(256), 0, st, a);
}

// A kernel's tile, and what a call on it takes: `start` us for the first workgroups of a CU and 1.5 for each further round of them; for every block of K that a workgroup
// (of the streaming kernels: a wavefront) walks, `alone` us or, where more workgroups share the CU, `shared` for each.
struct Fp8Kernel {
  int tokens, features, beside, walkers;      // beside: workgroups that a CU holds; walkers: wavefronts that share the blocks
  float start, alone, shared;
};
// Fitted to 14000 timings of 27 tiles in graphs, on 8 layers from 1024 x 1024 to 8192 x 28672 with 1 to 6000 tokens, whole and with K in 2 to 16 shares, weights not in the caches.  Up to
// 128 tokens the rule's pick is 0.3 % behind the best of all that were timed on average, 8 % at most; from 130 on 0.7 % and 8 %, and without the tiles of 96, 160, 192 and 224 tokens,
// which leave fewer CUs idle in the last round, 5.3 % and 27 % (1500 on 8192 x 8192 110 -> 101 us, 800 on 2000 x 5000 23 -> 19).
constexpr Fp8Kernel kFp8Kernels[] = {
    {16, 16, 2, 8, 3.644f, 0.306f, 0.369f},  {16, 32, 1, 8, 3.357f, 0.140f, 0.639f},  {32, 32, 1, 8, 3.500f, 0.885f, 0.414f},   {16, 128, 2, 1, 4.175f, 0.311f, 0.260f},
    {32, 128, 1, 1, 4.640f, 0.379f, 0.286f}, {64, 64, 2, 1, 4.963f, 0.354f, 0.255f},  {64, 128, 2, 1, 5.695f, 0.421f, 0.377f},
    {96, 128, 1, 1, 5.076f, 0.395f, 0.544f}, {128, 128, 1, 1, 5.864f, 0.626f, 0.091f}, {160, 128, 1, 1, 5.627f, 0.727f, 0.326f}, {96, 256, 1, 1, 5.722f, 0.826f, 0.045f},
    {128, 256, 1, 1, 7.185f, 0.942f, 0.152f}, {192, 256, 1, 1, 4.773f, 1.472f, 0.156f}, {224, 256, 1, 1, 5.354f, 1.552f, 0.361f}, {256, 256, 1, 1, 7.492f, 1.662f, 0.189f}};
constexpr int kFp8KernelCount = sizeof(kFp8Kernels) / sizeof(kFp8Kernels[0]);
constexpr int kFp8MaxSplits = 8;

struct Fp8Pick {
  int kernel, splits;
};
Fp8Pick pick_fp8(int tokens, int m, int k) {
  Fp8Pick best = {0, 1};
  float least = 3e38f;
  const int blocks = fp8_blocks(k);
  for (int i = 0; i < kFp8KernelCount; i++) {
    const Fp8Kernel& c = kFp8Kernels[i];
    // (The fitted costs would give 32 features a workgroup to large layers.  1 to 16 tokens in codes on 16 features and on 32, us, weights not in the caches: 4096 x 4096 6.1 to 6.6 and
    // 6.7 to 7.8, 4096 x 11008 11.6 to 12.6 and 13.2 to 14.3, 11008 x 4096 12.0 to 13.0 and 13.2 to 15.4, 4096 x 12288 12.3 to 13.4 and 13.5 to 14.7; on 8192 x 8192 14.0 to 15.5 and 13.9 to 14.1.)
    if (c.walkers > 1 && c.features > 16 && tokens <= 16) continue;
    const long tiles = ((tokens + c.tokens - 1L) / c.tokens) * ((m + c.features - 1L) / c.features);
    for (int splits = 1; splits <= kFp8MaxSplits; splits *= 2) {
      if (splits > 1 && (tiles * splits > 512 || blocks / splits < 8 || (c.walkers > 1 && (splits > 2 || tiles > 96)))) break;
      const int share = (blocks + splits - 1) / splits, walk = (share + c.walkers - 1) / c.walkers;
      const long deep = (tiles * splits + 255) / 256, rounds = deep / c.beside, rest = deep % c.beside;
      const float full = std::max(c.alone, c.shared * c.beside), part = rest ? std::max(c.alone, c.shared * rest) : 0.f;
      float us = c.start + 1.5f * (rounds + (rest > 0) - 1) + walk * (rounds * full + part);
      // the weights at 6.2 TB/s, and a part of what all tiles read from L2
      us = std::max(us, 3.f + ((float)m * k + (float)tokens * k) / 6.2e6f + 0.015e-6f * tiles * (c.tokens + c.features) * k);
      if (splits > 1) us += 2.f + 1e-6f * tokens * m * (splits + 1);
      if (us < least) least = us, best = {i, splits};
    }
  }
  return best;
}
// Rows of W lie a power of two apart, and walks in lockstep read the same few channels of HBM: in codes on 8192 x 28672, weights not in the caches, one token 52 us and spread 41, 64 56 and 48, 256
// 83 and 81; 16 on 4096 x 22016 24 and 19, on 4096 x 11008 13.2 and 12.6.  From 512 tokens on, on small layers and on weights that the Infinity Cache holds there is nothing to spread (512 131 and 131; 4096 x 4096
// 6.6 and 6.6; one token on 8192 x 28672 again and again 36.4 and 36.7).
bool fp8_rotates(int tokens, int m, int k) { return tokens <= 512 && (long)m * k >= (1L << 25); }

long fp8_units(const Fp8Args& a, int tokens, int features) { return ((a.m + features - 1L) / features) * ((a.tokens + tokens - 1L) / tokens) * a.splits; }

template <int NT, int TW, int F, int FW, int STAGES>
int launch_fp8_tile(const Fp8Args& a, hipStream_t st) {
  using Tile = Fp8Tile<NT, TW, F, FW, STAGES>;
  static_assert(Tile::kLdsBytes <= 163840, "");
  if (int e = grant_lds<fp8_tile_kernel<NT, TW, F, FW, STAGES>>(Tile::kLdsBytes, "fp8_tile_kernel")) return e;
  const long units = fp8_units(a, Tile::kTokens, Tile::kFeatures);
  if (units > 0x7ffffff0L) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "fp8_matmul: too many work units (%ld)", units);
  hipLaunchKernelGGL((fp8_tile_kernel<NT, TW, F, FW, STAGES>), dim3((unsigned)((units + 7) / 8 * 8)), dim3(Tile::kThreads), Tile::kLdsBytes, st, a);
  return check_launch("fp8_tile_kernel");
}
template <int NT, int F, int WAVES, int STAGES, class T = uint8_t>
int launch_fp8_stream(const Fp8Args& a, hipStream_t st) {
  using Tile = Fp8Stream<T, NT, F, WAVES, STAGES>;
  static_assert(Tile::kLdsBytes <= 163840, "");
  if (int e = grant_lds<fp8_stream_kernel<T, NT, F, WAVES, STAGES>>(Tile::kLdsBytes, "fp8_stream_kernel")) return e;
  const long units = fp8_units(a, Tile::kTokens, Tile::kFeatures);
  if (units > 0x7ffffff0L) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "fp8_matmul: too many work units (%ld)", units);
  hipLaunchKernelGGL((fp8_stream_kernel<T, NT, F, WAVES, STAGES>), dim3((unsigned)((units + 7) / 8 * 8)), dim3(Tile::kThreads), Tile::kLdsBytes, st, a);
  return check_launch("fp8_stream_kernel");
}
// in the order of kFp8Kernels
int launch_fp8(const Fp8Args& a, int kernel, hipStream_t st) {
  switch (kernel) {
    case 0: return launch_fp8_stream<1, 1, 8, 2>(a, st);
    case 1: return launch_fp8_stream<1, 2, 8, 2>(a, st);
    case 2: return launch_fp8_stream<2, 2, 8, 2>(a, st);
    case 3: return launch_fp8_tile<1, 1, 2, 4, 4>(a, st);
    case 4: return launch_fp8_tile<2, 1, 2, 4, 4>(a, st);
    case 5: return launch_fp8_tile<2, 2, 2, 2, 4>(a, st);
    case 6: return launch_fp8_tile<2, 2, 2, 4, 3>(a, st);
    case 7: return launch_fp8_tile<3, 2, 2, 4, 3>(a, st);
    case 8: return launch_fp8_tile<4, 2, 2, 4, 3>(a, st);
    case 9: return launch_fp8_tile<5, 2, 2, 4, 3>(a, st);
    case 10: return launch_fp8_tile<3, 2, 4, 4, 3>(a, st);
    case 11: return launch_fp8_tile<4, 2, 4, 4, 3>(a, st);
    case 12: return launch_fp8_tile<6, 2, 4, 4, 2>(a, st);
    case 13: return launch_fp8_tile<7, 2, 4, 4, 2>(a, st);
    default: return launch_fp8_tile<8, 2, 4, 4, 2>(a, st);
  }
}

// Up to 4 tokens in 16 bits on the streaming kernel: quantised on the way, without a launch of the quantiser and its scratch (one on 4096 x 4096 8.0 -> 6.4 us, a call from
// Python 7.8 -> 6.0; 4 on 4096 x 11008 13.4 -> 12.6).  Twice the rows take twice the vector instructions in every workgroup: 8 on 4096 x 11008 20.7.
constexpr int kFp8OnTheWay = 4;
bool fp8_at_once(int tokens, int x_type, const Fp8Pick& t) { return x_type != 2 && tokens <= kFp8OnTheWay && t.kernel == 0 && t.splits == 1; }

template <class T>
void launch_fp8_reduce(const Fp8Args& a, hipStream_t st) {
  const long results = (long)a.tokens * a.m;
  if (results % 4 == 0) hipLaunchKernelGGL((fp8_reduce_kernel<T, 4>), dim3((unsigned)((results / 4 + 255) / 256)), dim3(256), 0, st, a.partial, a.splits, results, static_cast<T*>(a.out));
  else hipLaunchKernelGGL((fp8_reduce_kernel<T, 1>), dim3((unsigned)((results + 255) / 256)), dim3(256), 0, st, a.partial, a.splits, results, static_cast<T*>(a.out));
}

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }
// activations in 16 bits: their codes and scales, a block's of all tokens adjacent
size_t fp8_codes_bytes(int tokens, int k) { return (size_t)tokens * k; }
size_t fp8_scales_bytes(int tokens, int k) { return round16(sizeof(float) * (size_t)tokens * fp8_blocks(k)); }

}  // namespace

extern "C" {

int triteia_hip_fp8_quantize(const void* x, long x_stride, int n, int k, int rows, void* codes, long codes_stride, void* scales, long scale_row, long scale_block,
                             int bf16, int dev, void* stream) {
  const char* what = "fp8_quantize";
  if (int e = check_fp8(what, n, k)) return e;
  if (rows != 1 && rows != 128) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: %d rows a scale: 1 or 128", what, rows);
  if (n == 0 || k == 0) return TRITEIA_HIP_OK;
  if (!x || !codes || !scales) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(x) || !aligned16(codes) || reinterpret_cast<uintptr_t>(scales) % 4 != 0 || !strides_ok({x_stride}, 2, 16) || !strides_ok({codes_stride}, 1, 8) ||
      codes_stride < k || scale_row < 0 || scale_block < 0)
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: rows of whole 16 bytes", what);
  if (fp8_groups(n, k, 1) > 0x7fffffffL) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: too many work units", what);
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  const Fp8QuantArgs a = {x, x_stride, static_cast<uint8_t*>(codes), codes_stride, static_cast<float*>(scales), scale_row, scale_block, n, k};
  return bf16 ? launch_fp8_quant<__bf16>(a, rows, static_cast<hipStream_t>(stream)) : launch_fp8_quant<_Float16>(a, rows, static_cast<hipStream_t>(stream));
}

int triteia_hip_fp8_values(const void* codes, long codes_stride, const void* scales, long scale_row, long scale_block, int rows, int n, int k, void* out, int type,
                           int dev, void* stream) {
  const char* what = "fp8_values";
  if (int e = check_fp8(what, n, k)) return e;
  if ((rows != 1 && rows != 128) || type < 0 || type > 2) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: %d rows a scale, type %d: 1 or 128, 0 to 2", what, rows, type);
  if (n == 0 || k == 0) return TRITEIA_HIP_OK;
  if (!codes || !scales || !out) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(codes) || !aligned16(out) || reinterpret_cast<uintptr_t>(scales) % 4 != 0 || !strides_ok({codes_stride}, 1, 8) || scale_row < 0 || scale_block < 0)
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: rows of whole 16 bytes", what);
  if (fp8_groups(n, k, 1) > 0x7fffffffL) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: too many work units", what);
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  const Fp8ValuesArgs a = {static_cast<const uint8_t*>(codes), codes_stride, static_cast<const float*>(scales), scale_row, scale_block, rows == 1 ? 0 : 7, out, n, k};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == 0) launch_fp8_values<_Float16>(a, st);
  else if (type == 1) launch_fp8_values<__bf16>(a, st);
  else launch_fp8_values<float>(a, st);
  return check_launch("fp8_values_kernel");
}

int triteia_hip_fp8_tile(int tokens, int m, int k) {
  if (tokens <= 0 || m <= 0 || k <= 0 || check_fp8("fp8_matmul", tokens, k) || m > kFp8Most) return 0;
  const Fp8Pick t = pick_fp8(tokens, m, k);
  return (t.splits * 1000 + kFp8Kernels[t.kernel].features) * 1000 + kFp8Kernels[t.kernel].tokens;
}

size_t triteia_hip_fp8_scratch_bytes(int tokens, int m, int k, int x_type) {
  if (tokens <= 0 || m <= 0 || k <= 0 || check_fp8("fp8_matmul", tokens, k) || m > kFp8Most) return 0;
  const Fp8Pick t = pick_fp8(tokens, m, k);
  const int splits = t.splits;
  return (x_type == 2 || fp8_at_once(tokens, x_type, t) ? 0 : fp8_codes_bytes(tokens, k) + fp8_scales_bytes(tokens, k)) + (splits > 1 ? sizeof(float) * (size_t)splits * tokens * m : 0);
}

int triteia_hip_fp8_matmul(const void* x, long x_stride, int x_type, const void* x_scale, long xs_token, long xs_block, const void* weight, long w_stride,
                           const void* w_scale, long ws_row, long ws_block, void* out, int out_type, int tokens, int m, int k, void* scratch, size_t scratch_bytes,
                           int dev, void* stream) {
  const char* what = "fp8_matmul";
  if (int e = check_fp8(what, tokens, k)) return e;
  if (m < 0 || m > kFp8Most) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d features: up to 2^24", what, m);
  if (x_type < 0 || x_type > 2 || out_type < 0 || out_type > 2) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: types %d and %d: 0 to 2", what, x_type, out_type);
  if (tokens == 0 || m == 0) return TRITEIA_HIP_OK;
  if (k == 0) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: rows without elements", what);
  if (!x || !weight || !w_scale || !out || (x_type == 2 && !x_scale)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(x) || !aligned16(weight) || !aligned16(out) || !strides_ok({x_stride}, x_type == 2 ? 1 : 2, 16) || !strides_ok({w_stride}, 1, 16) ||
      ws_row < 0 || ws_block < 0 || (x_type == 2 && (xs_token < 0 || xs_block < 0)) || w_stride > kFp8Most || x_stride > kFp8Most)
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: rows of x and of the weight start on 16 bytes and are up to 2^24 elements apart", what);
  const size_t need = triteia_hip_fp8_scratch_bytes(tokens, m, k, x_type);
  if (need && (!scratch || scratch_bytes < need || !aligned16(scratch)))
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: scratch must hold %zu bytes (got %zu), aligned to 16", what, need, scratch_bytes);
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  Fp8Args a = {};
  const Fp8Pick t = pick_fp8(tokens, m, k);
  const bool at_once = fp8_at_once(tokens, x_type, t);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  if (x_type == 2 || at_once) {
    a.x = static_cast<const uint8_t*>(x), a.x_stride = x_stride, a.xs = static_cast<const float*>(x_scale), a.xs_token = xs_token, a.xs_block = xs_block;
  } else {
    float* scales = reinterpret_cast<float*>(at + fp8_codes_bytes(tokens, k));
    const Fp8QuantArgs quant = {x, x_stride, at, k, scales, 1, tokens, tokens, k};
    if (int e = x_type == 1 ? launch_fp8_quant<__bf16>(quant, 1, st) : launch_fp8_quant<_Float16>(quant, 1, st)) return e;
    a.x = at, a.x_stride = k, a.xs = scales, a.xs_token = 1, a.xs_block = tokens;
    at += fp8_codes_bytes(tokens, k) + fp8_scales_bytes(tokens, k);
  }
  a.w = static_cast<const uint8_t*>(weight), a.w_stride = w_stride, a.ws = static_cast<const float*>(w_scale), a.ws_row = ws_row, a.ws_block = ws_block;
  a.out = out, a.type = out_type, a.tokens = tokens, a.m = m, a.k = k, a.splits = t.splits, a.rotate = fp8_rotates(tokens, m, k);
  a.partial = reinterpret_cast<float*>(at);
  if (at_once) return x_type == 1 ? launch_fp8_stream<1, 1, 8, 2, __bf16>(a, st) : launch_fp8_stream<1, 1, 8, 2, _Float16>(a, st);
  if (int e = launch_fp8(a, t.kernel, st)) return e;
  if (t.splits == 1) return TRITEIA_HIP_OK;
  if (out_type == 0) launch_fp8_reduce<_Float16>(a, st);
  else if (out_type == 1) launch_fp8_reduce<__bf16>(a, st);
  else launch_fp8_reduce<float>(a, st);
  return check_launch("fp8_reduce_kernel");
}

}  // extern "C"
