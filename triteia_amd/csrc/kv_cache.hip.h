// Rotary positions with the norms of queries and keys, the write of keys and values into a paged cache, and the read-back.
//
// A row is one head of one token, D elements.  Queries and keys, in 32 bits:
//   norm (where there is a weight)   x <- x * rsqrt(sum(x^2) / D + eps) * w
//   rotation of the first R elements (a, b) <- (a cos - b sin, b cos + a sin) with the pair (i, i + R / 2) or, interleaved,
//                                    (2 i, 2 i + 1), cos and sin of pair i from row `position` of a table [P, R / 2, 2]
// and one rounding to the type of the output.  A position outside the table gives a row of NaN (loud, and no access out of bounds).
// In a cache of 8 bits a row is codes and one scale: scale = max|x| / 127, code = x / scale to the nearest whole number (int8), or
// scale = max|x| / 448, code = x / scale to the nearest e4m3 (fp8).  Ties go to even.  A row of magnitudes below 1e-30 is zeros with scale 0; one that
// holds a NaN or an infinity gets the scale NaN, so that all of it reads back as NaN.
//
// Bound by memory, and for a decode batch by the launch and one round trip.  LPR lanes of 16 bytes hold a row (D / 8 rounded up to a power of
// two), a workgroup takes rows of one token, so cos, sin and the norms' weights are fetched once per lane and serve its U rows, whose loads
// are requested together.  The element across a rotated pair comes by a lane exchange of the packed values.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace triteia_hip {

// what a cache holds
enum CacheKind { kCacheSame = 0, kCacheInt8 = 1, kCacheFp8 = 2 };

template <class T> using kv8 = T __attribute__((ext_vector_type(8)));
typedef uint32_t kv_uint4 __attribute__((ext_vector_type(4)));
typedef float kv_float4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_uint2 __attribute__((ext_vector_type(2)));

// Where row (page, head, slot) of a cache lies: offsets in elements (bytes in an 8-bit cache); the elements of a row are adjacent.
struct CachePart {
  void* data;
  float* scale;                 // 8-bit caches: one per row
  long page, head, slot;        // strides of data
  long scale_page, scale_head, scale_slot;
};

struct RotaryArgs {
  const void *q, *k, *v;        // v null: none
  long q_token, q_head, k_token, k_head, v_token, v_head;
  void *q_out, *k_out;          // [tokens, heads, D]; k_out null: keys go to the cache
  int tokens, heads, kv_heads, dim, rot;
  const void* positions;        // null: no rotation
  const float* table;           // [limit, rot / 2, 2]
  long limit;
  const void *q_norm, *k_norm;  // null: none
  float eps;
  const void* slots;
  int positions64, slots64;
  int page_shift;
  long n_slots;                 // slots of the cache
  CachePart ck, cv;
};

__device__ __forceinline__ long index_at(const void* p, int wide, long i) {
  return wide ? static_cast<const int64_t*>(p)[i] : (long)static_cast<const int32_t*>(p)[i];
}

// 8 values as codes of the row's scale; inv = 1 / scale
template <int KIND>
__device__ __forceinline__ kv_uint2 codes_of(const float (&x)[8], float inv) {
  kv_uint2 c = {0, 0};
  if constexpr (KIND == kCacheInt8) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int v = (int)__builtin_amdgcn_fmed3f(__builtin_rintf(x[j] * inv), -127.f, 127.f);
      c[j / 4] |= (uint32_t)(v & 255) << (8 * (j % 4));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int w = 0;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = __builtin_amdgcn_fmed3f(x[4 * i + j] * inv, -448.f, 448.f);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
      c[i] = (uint32_t)w;
    }
  }
  return c;
}

template <int KIND>
__device__ __forceinline__ void values_of(kv_uint2 c, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if constexpr (KIND == kCacheInt8) {
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * i + j] = (float)(int)(int8_t)(c[i] >> (8 * j));
    } else {
      typedef float float2_t __attribute__((ext_vector_type(2)));
      const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
      x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = b.x, x[4 * i + 3] = b.y;
    }
  }
}

template <int N> struct KvControl { static constexpr int value = N; };
// The sum, or the largest, of a row's LPR lanes, in all of them: exchanges inside a quad, mirrors of 8 and of 16 lanes.
template <int LPR, class V, class F>
__device__ __forceinline__ V across_row(V v, F f) {
  auto dpp = [](V x, auto control) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value, 0xf, 0xf, true));
  };
  v = f(v, dpp(v, KvControl<0xb1>{}));
  v = f(v, dpp(v, KvControl<0x4e>{}));
  v = f(v, dpp(v, KvControl<0x141>{}));
  if constexpr (LPR >= 16) v = f(v, dpp(v, KvControl<0x140>{}));
  if constexpr (LPR >= 32) v = f(v, __builtin_bit_cast(V, __shfl_xor(__builtin_bit_cast(int, v), 16)));
  return v;
}

// One row of the cache: x[8] of each of the row's LPR lanes (`live`: the lane holds elements of the row).
template <class T, int KIND, int LPR>
__device__ __forceinline__ void cache_row(const CachePart& c, long page, long head, long slot, int e, bool live, const float (&x)[8]) {
  const long at = page * c.page + head * c.head + slot * c.slot + e;
  if constexpr (KIND == kCacheSame) {
    kv8<T> y;
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = (T)x[j];
    if (live) *reinterpret_cast<kv8<T>*>(static_cast<T*>(c.data) + at) = y;
  } else {
    uint32_t top = 0;           // (the bits of magnitudes order as the magnitudes do, infinity and NaN above them)
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
    if (!live) top = 0;
    top = across_row<LPR>(top, [](uint32_t p, uint32_t q) { return max(p, q); });
    const float most = __builtin_bit_cast(float, top);
    float scale = most / (KIND == kCacheInt8 ? 127.f : 448.f), inv = 1.f / scale;
    if (most < 1e-30f) scale = 0.f, inv = 0.f;
    kv_uint2 code = codes_of<KIND>(x, inv);
    if (top >= 0x7f800000u) scale = __builtin_nanf(""), code = kv_uint2{0, 0};
    if (live) *reinterpret_cast<kv_uint2*>(static_cast<uint8_t*>(c.data) + at) = code;
    if (e == 0) c.scale[page * c.scale_page + head * c.scale_head + slot * c.scale_slot] = scale;
  }
}

// grid (chunks of a token's rows, tokens), block 256.  A token's rows: heads of q, heads of k, heads of v.
template <class T, int KIND, int LPR, int U, bool NORM>
__global__ __launch_bounds__(256) void rotary_cache_kernel(RotaryArgs a, int interleaved) {
  constexpr int kRows = 256 / LPR;                 // rows of a pass
  const int lane = threadIdx.x % LPR, e = 8 * lane;
  const bool live = e < a.dim;
  const int n_rows = a.heads + a.kv_heads * (a.v ? 2 : 1);
  const int half = a.rot / 2;
  const bool turned = a.positions && e < a.rot, first = e < half;
  const int across = interleaved || !turned ? lane : first ? lane + half / 8 : lane - half / 8;
  const kv8<T> none = {0, 0, 0, 0, 0, 0, 0, 0};
  kv8<T> w[2], wx[2];             // norm weights of this lane's elements and of those across, for q and k
  if constexpr (NORM) {
#pragma unroll
    for (int n = 0; n < 2; n++) {
      const T* src = static_cast<const T*>(n ? a.k_norm : a.q_norm);
      w[n] = src && live ? *reinterpret_cast<const kv8<T>*>(src + e) : none;
      wx[n] = src && live ? *reinterpret_cast<const kv8<T>*>(src + 8 * across) : none;
      if (interleaved) wx[n] = __builtin_shufflevector(w[n], w[n], 1, 0, 3, 2, 5, 4, 7, 6);
    }
  }
  for (long t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    long page = 0, slot = -1;
    if (a.slots) {
      const long s = index_at(a.slots, a.slots64, t);
      if (s >= 0 && s < a.n_slots) page = s >> a.page_shift, slot = s & ((1 << a.page_shift) - 1);
    }
    // this lane's cos and sin: pairs e / 2 .. + 3 (interleaved) or e % (R / 2) .. + 7, minus in front of the sine of a pair's first element
    float c[8], s[8];
    if (turned) {
      const long p = index_at(a.positions, a.positions64, t);
      const bool inside = p >= 0 && p < a.limit;
      const int pair = interleaved ? e / 2 : first ? e : e - half;
      const kv_float4* row = reinterpret_cast<const kv_float4*>(a.table + (inside ? p : 0) * a.rot + 2 * pair);
      kv_float4 f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = i < 2 || !interleaved ? row[i] : kv_float4{0.f, 0.f, 0.f, 0.f};
      if (!inside) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = kv_float4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        c[j] = interleaved ? f[j / 4][j / 2 % 2 * 2] : f[j / 2][j % 2 * 2];
        s[j] = interleaved ? f[j / 4][j / 2 % 2 * 2 + 1] : f[j / 2][j % 2 * 2 + 1];
        if (interleaved ? j % 2 == 0 : first) s[j] = -s[j];
      }
    }
    for (int row0 = blockIdx.x * (kRows * U) + threadIdx.x / LPR; row0 < n_rows + (int)(threadIdx.x / LPR); row0 += gridDim.x * (kRows * U)) {
      kv8<T> x[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int r = row0 + u * kRows;
        const T* src = r < a.heads ? static_cast<const T*>(a.q) + t * a.q_token + r * a.q_head
                       : r < a.heads + a.kv_heads ? static_cast<const T*>(a.k) + t * a.k_token + (r - a.heads) * a.k_head
                                                  : static_cast<const T*>(a.v) + t * a.v_token + (r - a.heads - a.kv_heads) * a.v_head;
        x[u] = live && r < n_rows ? *reinterpret_cast<const kv8<T>*>(src + e) : none;
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int r = row0 + u * kRows;
        const bool is_q = r < a.heads, is_v = r >= a.heads + a.kv_heads;
        float y[8], o[8];          // own elements, and those across
        const kv_uint4 mine = __builtin_bit_cast(kv_uint4, x[u]);
        kv8<T> xo;
        if (interleaved) {
          xo = __builtin_shufflevector(x[u], x[u], 1, 0, 3, 2, 5, 4, 7, 6);
        } else {
          kv_uint4 other;
#pragma unroll
          for (int i = 0; i < 4; i++) other[i] = (uint32_t)__shfl((int)mine[i], across, LPR);
          xo = __builtin_bit_cast(kv8<T>, other);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = (float)x[u][j], o[j] = (float)xo[j];
        if constexpr (NORM) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; j++) sum = __builtin_fmaf(y[j], y[j], sum);
          sum = across_row<LPR>(sum, [](float p, float q) { return p + q; });
          if (!is_v && (is_q ? a.q_norm : a.k_norm) != nullptr) {
            const float f = __builtin_amdgcn_rsqf(sum / a.dim + a.eps);
            const kv8<T> own = is_q ? w[0] : w[1], far = is_q ? wx[0] : wx[1];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = y[j] * f * (float)own[j], o[j] = o[j] * f * (float)far[j];
          }
        }
        if (turned && !is_v) {
#pragma unroll
          for (int j = 0; j < 8; j++) y[j] = __builtin_fmaf(o[j], s[j], y[j] * c[j]);
        }
        if (r < n_rows && (is_q || a.k_out)) {
          kv8<T> out;
#pragma unroll
          for (int j = 0; j < 8; j++) out[j] = (T)y[j];
          T* dst = is_q ? static_cast<T*>(a.q_out) + (t * a.heads + r) * a.dim : static_cast<T*>(a.k_out) + (t * a.kv_heads + r - a.heads) * a.dim;
          if (live) *reinterpret_cast<kv8<T>*>(dst + e) = out;
        } else if (r < n_rows && slot >= 0) {
          cache_row<T, KIND, LPR>(is_v ? a.cv : a.ck, page, is_v ? r - a.heads - a.kv_heads : r - a.heads, slot, e, live, y);
        }
      }
    }
  }
}

struct CacheReadArgs {
  CachePart ck, cv;
  void *k_out, *v_out;           // [tokens, kv_heads, D]
  const void* slots;
  int slots64, tokens, kv_heads, dim, page_shift;
  long n_slots;
};

// grid (chunks of rows, 2: keys, values), block 256; rows in the order of the output (token, head).  A slot outside the cache gives zeros.
template <class T, int KIND, int LPR, int U>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadArgs a) {
  constexpr int kRows = 256 / LPR;
  const int e = 8 * (threadIdx.x % LPR);
  const CachePart& c = blockIdx.y ? a.cv : a.ck;
  T* out = static_cast<T*>(blockIdx.y ? a.v_out : a.k_out);
  const long n_rows = (long)a.tokens * a.kv_heads;
  const long row0 = (long)blockIdx.x * (kRows * U) + threadIdx.x / LPR;
  if (e >= a.dim) return;
  kv8<T> x[U];
  kv_uint2 code[U];
  float scale[U];
  bool inside[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long r = row0 + u * kRows;
    const uint32_t t = (uint32_t)((uint64_t)(r < n_rows ? r : n_rows - 1) / (uint32_t)a.kv_heads);
    const long head = (r < n_rows ? r : n_rows - 1) - (long)t * a.kv_heads;
    const long s = index_at(a.slots, a.slots64, t);
    inside[u] = s >= 0 && s < a.n_slots;
    const long page = inside[u] ? s >> a.page_shift : 0, slot = inside[u] ? s & ((1 << a.page_shift) - 1) : 0;
    const long at = page * c.page + head * c.head + slot * c.slot + e;
    if constexpr (KIND == kCacheSame) {
      x[u] = *reinterpret_cast<const kv8<T>*>(static_cast<const T*>(c.data) + at);
    } else {
      code[u] = *reinterpret_cast<const kv_uint2*>(static_cast<const uint8_t*>(c.data) + at);
      scale[u] = c.scale[page * c.scale_page + head * c.scale_head + slot * c.scale_slot];
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long r = row0 + u * kRows;
    if (r >= n_rows) return;
    if constexpr (KIND != kCacheSame) {
      float y[8];
      values_of<KIND>(code[u], y);
#pragma unroll
      for (int j = 0; j < 8; j++) x[u][j] = (T)(y[j] * scale[u]);
    }
    if (!inside[u]) x[u] = kv8<T>{0, 0, 0, 0, 0, 0, 0, 0};
    *reinterpret_cast<kv8<T>*>(out + r * a.dim + e) = x[u];
  }
}

}  // namespace triteia_hip
