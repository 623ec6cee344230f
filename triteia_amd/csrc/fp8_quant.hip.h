// Values in 8 bits with a scale for each block: x [n, k] in blocks of 1 x 128 (activations) or 128 x 128 (weights), the last ones smaller.
//   a = max|x| over the block, scale = a / 448, code = x / scale to the nearest e4m3, ties to even; value = code * scale
// A block of magnitudes below 1e-30 is zeros with scale 0; one that holds a NaN or an infinity gets the scale NaN, so that all of it
// reads back as NaN.  Scale and quotient are rounded as 32-bit divisions round.
//
// Bound by memory: 16 lanes of 16 bytes hold a row of a block, so that a maximum over it is four lane moves.  8000 x 8192 in bf16, four tensors in turn, 38 us and back 38 (5.2 TB/s; a
// large copy reaches 5.3), the same one again, parts of which the caches hold, 32 to 35 and 29; 11008 x 4096 in blocks of 128 x 128 again and again 23 and 20, 13 x 4096 2.3 and 2.2, which is a launch.
#pragma once
#include "kv_cache.hip.h"

namespace triteia_hip {

constexpr int kFp8Block = 128;

struct Fp8QuantArgs {
  const void* x;          // [n, k] of T
  long x_stride;
  uint8_t* codes;         // [n, k]
  long codes_stride;
  float* scales;
  long scale_row, scale_block;     // strides; a row is n's, or 128 of them
  int n, k;               // k a multiple of 16
};

// the scale of a block whose largest magnitude has these bits, and 1 / scale
__device__ __forceinline__ void fp8_scale(uint32_t top, float* scale, float* inv) {
  const float most = __builtin_bit_cast(float, top);
  *scale = most / 448.f, *inv = 1.f / *scale;
  if (most < 1e-30f) *scale = 0.f, *inv = 0.f;
  if (top >= 0x7f800000u) *scale = __builtin_nanf("");
}
template <class T>
__device__ __forceinline__ uint32_t fp8_top(const kv8<T>& v, float (&x)[8]) {
  uint32_t top = 0;         // (the bits of magnitudes order as the magnitudes do, infinity and NaN above them)
#pragma unroll
  for (int j = 0; j < 8; j++) {
    x[j] = (float)v[j];
    top = max(top, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
  }
  return top;
}

// 8 values of a row of a block, which 16 lanes hold: their codes and the block's scale
template <class T>
__device__ __forceinline__ kv_uint2 fp8_quantised(const kv8<T>& v, float* scale) {
  float x[8], inv;
  const uint32_t top = across_row<16>(fp8_top<T>(v, x), [](uint32_t p, uint32_t q) { return max(p, q); });
  fp8_scale(top, scale, &inv);
  const kv_uint2 code = codes_of<kCacheFp8>(x, *scale, inv);
  return top >= 0x7f800000u ? kv_uint2{0, 0} : code;
}

// Rows by themselves.  A workgroup takes 16 rows x U blocks.  1-D grid (row groups x block groups, block groups fastest), block 256
template <class T, int U>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(Fp8QuantArgs a) {
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block, across = (blocks + U - 1) / U;
  const int rows = blockIdx.x / across, b0 = (blockIdx.x - rows * across) * U;
  const int lane = threadIdx.x & 15;
  const long row = 16L * rows + (threadIdx.x >> 4);
  kv8<T> v[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int e = kFp8Block * (b0 + u) + 8 * lane;
    v[u] = kv8<T>{0, 0, 0, 0, 0, 0, 0, 0};
    if (row < a.n && e < a.k) v[u] = *reinterpret_cast<const kv8<T>*>(static_cast<const T*>(a.x) + row * a.x_stride + e);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    float scale;
    const kv_uint2 code = fp8_quantised<T>(v[u], &scale);
    const int e = kFp8Block * (b0 + u) + 8 * lane;
    if (row >= a.n || e >= a.k) continue;
    *reinterpret_cast<kv_uint2*>(a.codes + row * a.codes_stride + e) = code;
    if (lane == 0) a.scales[row * a.scale_row + (b0 + u) * a.scale_block] = scale;
  }
}

// 128 rows a scale: a workgroup takes a block.  1-D grid (row groups x blocks, blocks fastest), block 256
template <class T>
__global__ __launch_bounds__(256) void fp8_quant_tiles_kernel(Fp8QuantArgs a) {
  __shared__ uint32_t tops[4];
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block;
  const int rows = blockIdx.x / blocks, b = blockIdx.x - rows * blocks;
  const int e = kFp8Block * b + 8 * (threadIdx.x & 15);
  const long row0 = 128L * rows + (threadIdx.x >> 4);
  kv8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    v[i] = kv8<T>{0, 0, 0, 0, 0, 0, 0, 0};
    if (row0 + 16 * i < a.n && e < a.k) v[i] = *reinterpret_cast<const kv8<T>*>(static_cast<const T*>(a.x) + (row0 + 16 * i) * a.x_stride + e);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float x[8];
    top = max(top, fp8_top<T>(v[i], x));
  }
  top = across_row<32>(top, [](uint32_t p, uint32_t q) { return max(p, q); });
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  float scale, inv;
  fp8_scale(top, &scale, &inv);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float x[8];
    fp8_top<T>(v[i], x);
    kv_uint2 code = codes_of<kCacheFp8>(x, scale, inv);
    if (top >= 0x7f800000u) code = kv_uint2{0, 0};
    if (row0 + 16 * i < a.n && e < a.k) *reinterpret_cast<kv_uint2*>(a.codes + (row0 + 16 * i) * a.codes_stride + e) = code;
  }
  if (threadIdx.x == 0) a.scales[rows * a.scale_row + b * a.scale_block] = scale;
}

struct Fp8ValuesArgs {
  const uint8_t* codes;
  long codes_stride;
  const float* scales;
  long scale_row, scale_block;
  int row_shift;          // rows of a scale: 2^row_shift
  void* out;              // [n, k] of T
  int n, k;
};

// A workgroup takes 16 rows x one block (four of them, as above: 8000 x 8192 28.9 -> 29.6 us).
template <class T>
__global__ __launch_bounds__(256) void fp8_values_kernel(Fp8ValuesArgs a) {
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block;
  const int rows = blockIdx.x / blocks, b = blockIdx.x - rows * blocks;
  const long row = 16L * rows + (threadIdx.x >> 4);
  const int e = kFp8Block * b + 8 * (threadIdx.x & 15);
  if (row >= a.n || e >= a.k) return;
  float x[8];
  values_of<kCacheFp8>(*reinterpret_cast<const kv_uint2*>(a.codes + row * a.codes_stride + e), x);
  const float scale = a.scales[(row >> a.row_shift) * a.scale_row + b * a.scale_block];
  kv8<T> y;
#pragma unroll
  for (int j = 0; j < 8; j++) y[j] = (T)(x[j] * scale);
  *reinterpret_cast<kv8<T>*>(static_cast<T*>(a.out) + row * a.k + e) = y;
}

}  // namespace triteia_hip
