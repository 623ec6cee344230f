// Rotary positions with the norms of queries and keys, the write of keys and values into a paged cache, and the read-back.
//
// A row is one head of one token, D elements.  Queries and keys, in 32 bits:
//   norm (where there is a weight)   x <- x * rsqrt(sum(x^2) / D + eps) * w
//   rotation of the first R elements (a, b) <- (a cos - b sin, b cos + a sin) with the pair (i, i + R / 2) or, interleaved,
//                                    (2 i, 2 i + 1), cos and sin of pair i from row `position` of a table [P, R / 2, 2]
// and one rounding to the type of the output.  A position outside the table gives NaN in the elements that are rotated (loud, and no access out of bounds).
// In a cache of 8 bits a row is codes and one scale: scale = max|x| / 127, code = x / scale to the nearest whole number (int8), or
// scale = max|x| / 448, code = x / scale to the nearest e4m3 (fp8).  Ties go to even.  A row of magnitudes below 1e-30 is zeros with scale 0; one that
// holds a NaN or an infinity gets the scale NaN, so that all of it reads back as NaN.
//
// Bound by memory, and for a decode batch by the launch and one round trip.  LPR lanes of 16 bytes hold a row (D / 8 rounded up to a power of
// two); a workgroup takes rows of one token, so cos, sin and the norms' weights are fetched once per lane and serve all its rows.
// Measured: 8000 tokens of 40 + 40 heads of 128 in bf16 with norms 63 - 66 us (328 MB, 5.0 - 5.2 TB/s, what a copy reaches); 2000 tokens of 64 + 8 + 8 heads
// into an int8 cache 21 us (78 MB, 3.7 TB/s: position -> table row -> six passes, one after the other), 18 into a bf16 one; 64 tokens of 32 + 32 + 32 heads 4.4 us; 20000
// tokens of 32 heads read back from e4m3 98 - 103 us a call (497 MB, 4.8 - 5.1 TB/s).
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
  float eps, inv_dim;
  const void* slots;
  int positions64, slots64;
  int page_shift;
  long n_slots;                 // slots of the cache
  CachePart ck, cv;
};

__device__ __forceinline__ long index_at(const void* p, int wide, long i) {
  return wide ? static_cast<const int64_t*>(p)[i] : (long)static_cast<const int32_t*>(p)[i];
}
// The same for an index that all lanes share, from memory that the kernel does not write: a scalar load.
__device__ __forceinline__ long shared_index_at(const void* p, int wide, long i) {
  typedef const __attribute__((address_space(4))) int64_t* Wide;
  typedef const __attribute__((address_space(4))) int32_t* Narrow;
  return wide ? reinterpret_cast<Wide>(reinterpret_cast<uintptr_t>(p))[i] : (long)reinterpret_cast<Narrow>(reinterpret_cast<uintptr_t>(p))[i];
}

// 8 values as codes of the row's scale; inv = 1 / scale.  The quotient is x / scale as 32 bits round it, by one correction of x * inv: without it one value in
// 20000 takes the code on the other side of the middle.
template <int KIND>
__device__ __forceinline__ kv_uint2 codes_of(const float (&x)[8], float scale, float inv) {
  kv_uint2 c = {0, 0};
  float quotient[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float y = x[j] * inv;
    quotient[j] = __builtin_fmaf(__builtin_fmaf(-y, scale, x[j]), inv, y);
  }
  if constexpr (KIND == kCacheInt8) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int v = (int)__builtin_amdgcn_fmed3f(__builtin_rintf(quotient[j]), -127.f, 127.f);
      c[j / 4] |= (uint32_t)(v & 255) << (8 * (j % 4));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int w = 0;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = __builtin_amdgcn_fmed3f(quotient[4 * i + j], -448.f, 448.f);
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
    kv_uint2 code = codes_of<KIND>(x, scale, inv);
    if (top >= 0x7f800000u) scale = __builtin_nanf(""), code = kv_uint2{0, 0};
    if (live) *reinterpret_cast<kv_uint2*>(static_cast<uint8_t*>(c.data) + at) = code;
    if (e == 0) c.scale[page * c.scale_page + head * c.scale_head + slot * c.scale_slot] = scale;
  }
}

// Passes of 256 / LPR rows over a token's heads of q, of k and of v, none of two kinds.
struct RotaryPasses {
  int q, k, v;
  __host__ __device__ RotaryPasses(const RotaryArgs& a, int rows) : q((a.heads + rows - 1) / rows), k((a.kv_heads + rows - 1) / rows), v(a.v ? k : 0) {}
  __host__ __device__ int all() const { return q + k + v; }
};

__device__ __forceinline__ void kv_to_lds(const void* src, void* dst) {      // 16 bytes a lane, to dst + 16 lane
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// grid (passes of a token / U, tokens), block 256; with fewer workgroups than tokens they walk them.  The rows of U passes are requested together, by
// direct loads to LDS, and worked on one after the other: held in registers the compiler runs them side by side in 120 to 220 of these, and the
// wavefronts that are missing then cost more (8000 tokens of 80 heads with norms 114 us, a row at a time 96, this 65; three passes instead of six 72).  A
// wavefront reads what it has loaded itself, the element across a pair from its neighbour's place.  What does not depend on the row is multiplied
// first: cos and sin with the norm's weights, once for q and once for k of a token.  Indices come by scalar loads, ahead of everything.
template <class T, int KIND, int LPR, int U, bool NORM>
__global__ __launch_bounds__(256) void rotary_cache_kernel(RotaryArgs a, int interleaved) {
  constexpr int kRows = 256 / LPR;                 // rows of a pass
  const int lane = threadIdx.x % LPR, e = 8 * lane, row = threadIdx.x / LPR;
  const bool live = e < a.dim;
  const RotaryPasses passes(a, kRows);
  const int half = a.rot / 2;
  const bool turned = a.positions && e < a.rot, first = e < half;
  const int across = interleaved || !turned ? lane : first ? lane + half / 8 : lane - half / 8;
  const int pair = interleaved ? e / 2 : first ? e : e - half;      // of this lane's first element
  const kv8<T> none = {0, 0, 0, 0, 0, 0, 0, 0};
  __shared__ kv8<T> xs[U][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), beside = (int)threadIdx.x - lane + across;
  __shared__ kv8<T> weights[2][LPR];
  bool settled = !NORM;
  for (long t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const long position = a.positions ? shared_index_at(a.positions, a.positions64, t) : 0, to = a.slots ? shared_index_at(a.slots, a.slots64, t) : -1;
    auto request = [&](int pass, int u) {
      const T* src;
      int head = row;
      long step;
      if (pass < passes.q) src = static_cast<const T*>(a.q) + t * a.q_token, step = a.q_head, head += pass * kRows;
      else if (pass < passes.q + passes.k) src = static_cast<const T*>(a.k) + t * a.k_token, step = a.k_head, head += (pass - passes.q) * kRows;
      else src = static_cast<const T*>(a.v) + t * a.v_token, step = a.v_head, head += (pass - passes.q - passes.k) * kRows;
      if (live && head < (pass < passes.q ? a.heads : a.kv_heads)) kv_to_lds(src + head * step + e, &xs[u][64 * wave]);
    };
    const int pass0 = blockIdx.x * U, n = min(U, passes.all() - pass0);
    for (int u = 0; u < n; u++) request(pass0 + u, u);
    kv_float4 f[4];                 // cos and sin of this lane's pairs: 4 of them (interleaved) or 8
    const bool inside = position >= 0 && position < a.limit;
    if (turned) {
      const kv_float4* at = reinterpret_cast<const kv_float4*>(a.table + (inside ? position : 0) * a.rot + 2 * pair);
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = at[i < 2 || !interleaved ? i : 0];
    }
    if (!settled) {                 // (behind the requests of the first token)
      for (int i = threadIdx.x; i < 2 * LPR; i += 256) {
        const T* src = static_cast<const T*>(i < LPR ? a.q_norm : a.k_norm);
        if (src && 8 * (i % LPR) < a.dim) weights[i / LPR][i % LPR] = *reinterpret_cast<const kv8<T>*>(src + 8 * (i % LPR));
      }
      __syncthreads();
      settled = true;
    }
    const bool kept = to >= 0 && to < a.n_slots;
    const long page = kept ? to >> a.page_shift : 0, slot = kept ? to & ((1 << a.page_shift) - 1) : -1;
    float c[8], s[8];               // what this lane's elements and those across are multiplied by
    int kind = -1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int u = 0; u < n; u++) {
      const int pass = pass0 + u;
      const kv8<T> x = live ? xs[u][threadIdx.x] : none;
      const int now = pass < passes.q ? 0 : pass < passes.q + passes.k ? 1 : 2;
      const int head = row + kRows * (pass - (now == 0 ? 0 : now == 1 ? passes.q : passes.q + passes.k));
      const T* weight = static_cast<const T*>(now == 0 ? a.q_norm : a.k_norm);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = (float)x[j];
      if (now != 2) {
        if (now != kind) {
          kind = now;
          if (turned && interleaved) {
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = f[j / 4][j / 2 % 2 * 2], s[j] = j % 2 ? f[j / 4][j / 2 % 2 * 2 + 1] : -f[j / 4][j / 2 % 2 * 2 + 1];
          } else if (turned) {
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = f[j / 2][j % 2 * 2], s[j] = first ? -f[j / 2][j % 2 * 2 + 1] : f[j / 2][j % 2 * 2 + 1];
          } else {
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = 1.f, s[j] = 0.f;
          }
          if (turned && !inside) {
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = __builtin_nanf("");
          }
          if (NORM && weight && live) {
            const kv8<T> w = weights[now][lane], wx = weights[now][across], wi = __builtin_shufflevector(w, w, 1, 0, 3, 2, 5, 4, 7, 6);
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] *= (float)w[j], s[j] *= interleaved ? (float)wi[j] : (float)wx[j];
          }
        }
        float z[8];
        if (interleaved) {
#pragma unroll
          for (int j = 0; j < 8; j++) z[j] = turned ? y[j ^ 1] : 0.f;
        } else {
          const kv8<T> far = turned ? xs[u][beside] : none;                // (zero times an infinity would be a NaN)
#pragma unroll
          for (int j = 0; j < 8; j++) z[j] = (float)far[j];
        }
        float norm = 1.f;
        if (NORM && weight) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; j++) sum = __builtin_fmaf(y[j], y[j], sum);
          sum = across_row<LPR>(sum, [](float p, float q) { return p + q; });
          norm = __builtin_amdgcn_rsqf(__builtin_fmaf(sum, a.inv_dim, a.eps));
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
          y[j] = __builtin_fmaf(z[j], s[j], y[j] * c[j]);
          if (NORM && weight) y[j] *= norm;
        }
      }
      if (now == 0 || a.k_out) {
        kv8<T> out;
#pragma unroll
        for (int j = 0; j < 8; j++) out[j] = (T)y[j];
        T* dst = now == 0 ? static_cast<T*>(a.q_out) + (t * a.heads + head) * a.dim : static_cast<T*>(a.k_out) + (t * a.kv_heads + head) * a.dim;
        if (live && head < (now == 0 ? a.heads : a.kv_heads)) *reinterpret_cast<kv8<T>*>(dst + e) = out;
      } else if (slot >= 0 && head < a.kv_heads) {
        cache_row<T, KIND, LPR>(now == 2 ? a.cv : a.ck, page, head, slot, e, live, y);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                      // (the next token's rows go where these were read)
  }
}

struct CacheReadArgs {
  CachePart ck, cv;
  void *k_out, *v_out;           // [tokens, kv_heads, D]
  const void* slots;
  int slots64, tokens, kv_heads, dim, page_shift;
  long n_slots;
};

// grid (tiles, 2: keys, values), block 256.  A tile is 4 heads of adjacent tokens, whose rows of a head lie side by side in a page (in the order of the
// output, all heads of two tokens, 20000 tokens of 32 heads took 113 us instead of 105; stores past the caches made no difference at any size, 102.3 and
// 102.0).  A slot outside the cache gives zeros.
template <class T, int KIND, int LPR, int U>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadArgs a) {
  constexpr int kRows = 256 / LPR, kTokens = kRows * U / 4;
  const int e = 8 * (threadIdx.x % LPR);
  const CachePart& c = blockIdx.y ? a.cv : a.ck;
  T* out = static_cast<T*>(blockIdx.y ? a.v_out : a.k_out);
  const uint32_t heads4 = ((uint32_t)a.kv_heads + 3) / 4, tile = blockIdx.x / heads4;
  const int row0 = threadIdx.x / LPR;
  const int head = 4 * (int)(blockIdx.x - tile * heads4) + row0 % 4;
  if (e >= a.dim || head >= a.kv_heads) return;
  const long t0 = (long)tile * kTokens + row0 / 4;
  kv8<T> x[U];
  kv_uint2 code[U];
  float scale[U];
  bool inside[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long t = t0 + u * (kRows / 4);
    const long s = t < a.tokens ? index_at(a.slots, a.slots64, t) : -1;
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
    const long t = t0 + u * (kRows / 4);
    if (t >= a.tokens) return;
    if constexpr (KIND != kCacheSame) {
      float y[8];
      values_of<KIND>(code[u], y);
#pragma unroll
      for (int j = 0; j < 8; j++) x[u][j] = (T)(y[j] * scale[u]);
    }
    if (!inside[u]) x[u] = kv8<T>{0, 0, 0, 0, 0, 0, 0, 0};
    *reinterpret_cast<kv8<T>*>(out + (t * a.kv_heads + head) * a.dim + e) = x[u];
  }
}

}  // namespace triteia_hip
