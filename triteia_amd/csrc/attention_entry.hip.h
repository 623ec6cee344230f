// C entry points of the attention side (kv_cache.hip.h, attention_plan.hip.h, paged_attention.hip.h); part of triteia_hip.hip.
#pragma once

namespace {

// Workgroups that walk a large batch's tokens: the five that a CU's registers hold.  (One for every token left the last round half empty: 2000 tokens of 64 + 8 + 8
// heads into an int8 cache 22.9 us, 20.9 with 1280, 21.9 with 1536, 23.5 with 768; 8000 of 40 + 40 63.7, 62.8, 70.7, 69.5.)
constexpr int kRotaryWalks = 1280;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// rows of `dim` adjacent elements of `size` bytes, `align` of them at a time
bool strides_ok(std::initializer_list<long> strides, long size, long align) {
  for (long s : strides)
    if (s < 0 || s * size % align != 0) return false;
  return true;
}

struct CacheGeometry {
  int n_pages, kv_heads, page_shift, dim, kind;
};

int check_cache(const char* what, const CachePart& k, const CachePart& v, int n_pages, int kv_heads, int page, int dim, int kind) {
  if (kind < kCacheSame || kind > kCacheFp8) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: cache kind %d: 0 (16 bits), 1 (int8) or 2 (e4m3)", what, kind);
  if (n_pages < 1 || kv_heads < 1 || page < 16 || page > 1024 || (page & (page - 1)) != 0)
    return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: a cache of %d pages, %d heads, %d tokens a page: pages of 16, 32, .. 1024 tokens, one page and head at least", what,
                n_pages, kv_heads, page);
  const long size = kind == kCacheSame ? 2 : 1, align = kind == kCacheSame ? 16 : 8;
  for (const CachePart* p : {&k, &v}) {
    if (!p->data || (kind != kCacheSame && !p->scale)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null cache or scale pointer", what);
    if (!aligned16(p->data) || !strides_ok({p->page, p->head, p->slot}, size, align))
      return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a cache's rows need %ld-byte alignment", what, align);
  }
  (void)dim;
  return TRITEIA_HIP_OK;
}

int page_shift_of(int page) { return __builtin_ctz((unsigned)page); }

CachePart cache_part(const void* data, const void* scale, const long* strides, const long* scale_strides) {
  CachePart p = {};
  p.data = const_cast<void*>(data), p.scale = const_cast<float*>(static_cast<const float*>(scale));
  if (strides) p.page = strides[0], p.head = strides[1], p.slot = strides[2];
  if (scale_strides) p.scale_page = scale_strides[0], p.scale_head = scale_strides[1], p.scale_slot = scale_strides[2];
  return p;
}

template <class T, int KIND, int LPR, int U>
void launch_rotary(const RotaryArgs& a, int interleaved, hipStream_t stream) {
  const int chunks = (RotaryPasses(a, 256 / LPR).all() + U - 1) / U, walks = (kRotaryWalks + chunks - 1) / chunks;
  const dim3 grid(chunks, U == 1 || a.tokens < walks ? a.tokens : walks);
  if (a.q_norm || a.k_norm) hipLaunchKernelGGL((rotary_cache_kernel<T, KIND, LPR, U, true>), grid, dim3(256), 0, stream, a, interleaved);
  else hipLaunchKernelGGL((rotary_cache_kernel<T, KIND, LPR, U, false>), grid, dim3(256), 0, stream, a, interleaved);
}
template <class T, int KIND, int LPR>
void launch_rotary(const RotaryArgs& a, int interleaved, hipStream_t stream) {
  // small batches: a workgroup for every pass of 256 lanes; once that would be more than two for every CU, one for six of them
  if ((long)RotaryPasses(a, 256 / LPR).all() * a.tokens > 512) launch_rotary<T, KIND, LPR, 6>(a, interleaved, stream);
  else launch_rotary<T, KIND, LPR, 1>(a, interleaved, stream);
}
template <class T, int KIND>
void launch_rotary_lanes(const RotaryArgs& a, int interleaved, hipStream_t stream) {
  if (a.dim <= 64) launch_rotary<T, KIND, 8>(a, interleaved, stream);
  else if (a.dim <= 128) launch_rotary<T, KIND, 16>(a, interleaved, stream);
  else launch_rotary<T, KIND, 32>(a, interleaved, stream);
}

template <class T, int KIND, int LPR, int U>
void launch_read_tiles(const CacheReadArgs& a, hipStream_t stream) {
  constexpr long tokens = 256 / LPR * U / 4;
  const dim3 grid((unsigned)((a.tokens + tokens - 1) / tokens * ((a.kv_heads + 3) / 4)), 2);
  hipLaunchKernelGGL((cache_read_kernel<T, KIND, LPR, U>), grid, dim3(256), 0, stream, a);
}
template <class T, int KIND>
void launch_read(const CacheReadArgs& a, hipStream_t stream) {
  if (a.dim <= 64) launch_read_tiles<T, KIND, 8, 2>(a, stream);
  else if (a.dim <= 128) launch_read_tiles<T, KIND, 16, 2>(a, stream);
  else launch_read_tiles<T, KIND, 32, 2>(a, stream);
}

// the activations' type and what the cache holds, as template arguments
template <class F>
void by_types(int bf16, int kind, F f) {
  if (bf16) {
    if (kind == kCacheSame) f.template operator()<__bf16, kCacheSame>();
    else if (kind == kCacheInt8) f.template operator()<__bf16, kCacheInt8>();
    else f.template operator()<__bf16, kCacheFp8>();
  } else {
    if (kind == kCacheSame) f.template operator()<_Float16, kCacheSame>();
    else if (kind == kCacheInt8) f.template operator()<_Float16, kCacheInt8>();
    else f.template operator()<_Float16, kCacheFp8>();
  }
}

struct RotaryLaunch {
  const RotaryArgs& a;
  int interleaved;
  hipStream_t stream;
  template <class T, int KIND> void operator()() { launch_rotary_lanes<T, KIND>(a, interleaved, stream); }
};
struct ReadLaunch {
  const CacheReadArgs& a;
  hipStream_t stream;
  template <class T, int KIND> void operator()() { launch_read<T, KIND>(a, stream); }
};

template <class T, int KIND, int D>
void launch_attend(AttendArgs a, const AttnLayout& layout, float* scratch, long table_tokens, hipStream_t stream) {
  int joins = 0;
  for (int which = 0; which < 2; which++) {
    const AttnList& l = a.list[which] = layout.list[which];
    // (contexts that a table of so few tokens can hold are not cut)
    if (table_tokens > (long)l.min_blocks * kAttnBlock) joins += l.max_joins * a.kv_heads * (l.rows / (1024 / D));
    a.part_o[which] = scratch;
    a.part_ml[which] = scratch + (long)l.max_parts * a.kv_heads * l.rows * D;
    scratch = a.part_ml[which] + 2L * l.max_parts * a.kv_heads * l.rows;
  }
  a.joined = joins > 0;
  const dim3 grid((unsigned)((long)(a.list[0].max_items + a.list[1].max_items) * a.kv_heads));
  if (a.list[1].max_items > 0) hipLaunchKernelGGL((attend_mixed_kernel<T, KIND, D>), grid, dim3(256), 0, stream, a);
  else if (a.list[0].rows == 16 && a.list[0].waves == 8) hipLaunchKernelGGL((attend_rows_kernel<T, KIND, D, 1, 8>), grid, dim3(512), 0, stream, a);
  else if (a.list[0].rows == 16) hipLaunchKernelGGL((attend_rows_kernel<T, KIND, D, 1, 4>), grid, dim3(256), 0, stream, a);
  else if (a.list[0].waves == 8) hipLaunchKernelGGL((attend_rows_kernel<T, KIND, D, 2, 8>), grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL((attend_rows_kernel<T, KIND, D, 2, 4>), grid, dim3(256), 0, stream, a);
  if (joins > 0) hipLaunchKernelGGL((attend_join_kernel<T, D>), dim3(joins < kAttnJoiners ? joins : kAttnJoiners), dim3(256), 0, stream, a);
}
struct AttendLaunch {
  const AttendArgs& a;
  const AttnLayout& layout;
  float* scratch;
  long table_tokens;
  int dim;
  hipStream_t stream;
  template <class T, int KIND> void operator()() {
    if (dim == 64) launch_attend<T, KIND, 64>(a, layout, scratch, table_tokens, stream);
    else launch_attend<T, KIND, 128>(a, layout, scratch, table_tokens, stream);
  }
};

int check_batch(const char* what, int n_seqs, int n_tokens, int heads, int kv_heads, int max_q, int causal, int window) {
  if (n_seqs < 0 || n_seqs > kAttnMaxSeqs || n_tokens < 0 || n_tokens > (1 << 24) || max_q < 0 || window < 0)
    return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d sequences, %d tokens, at most %d of one, window %d: up to %d sequences and 2^24 tokens", what, n_seqs, n_tokens, max_q,
                window, kAttnMaxSeqs);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 1024)
    return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d heads over %d heads of the cache: a multiple, up to 1024", what, heads, kv_heads);
  if ((long)n_tokens * (heads / kv_heads) > (1L << 30)) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d tokens of %d heads are too many", what, n_tokens, heads);
  if (window > 0 && !causal) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a window needs causal", what);
  const AttnLayout l = attn_layout(n_seqs, n_tokens, heads, kv_heads, max_q, causal, window);
  for (const AttnList& x : l.list)
    if ((long)x.max_items * kv_heads > 0x3fffffffL || x.max_items < 0)
      return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: too many tiles", what);
  return TRITEIA_HIP_OK;
}

}  // namespace

extern "C" {

int triteia_hip_rotary_cache(const void* q, long q_token, long q_head, const void* k, long k_token, long k_head, const void* v, long v_token, long v_head,
                             void* q_out, void* k_out, int tokens, int heads, int kv_heads, int dim, int rot, const void* positions, int positions64,
                             const void* table, long limit, int interleaved, const void* q_norm, const void* k_norm, float eps, const void* slots, int slots64,
                             const void* cache_k, const void* cache_v, const void* k_scale, const void* v_scale, const long* strides, int n_pages, int page,
                             int kind, int bf16, int dev, void* stream) {
  const char* what = "rotary_cache";
  if (tokens < 0 || heads < 0 || kv_heads < 0 || heads > 65536 || kv_heads > 65536) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d tokens, %d + %d heads", what, tokens, heads, kv_heads);
  if (dim < 8 || dim > 256 || dim % 8 != 0) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: heads of %d elements: a multiple of 8 up to 256", what, dim);
  if (positions && (rot < 16 || rot > dim || rot % 16 != 0 || !table || limit < 1))
    return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: %d of %d elements rotated: a multiple of 16, and a table with a row at least", what, rot, dim);
  const bool to_cache = strides != nullptr;
  if (!to_cache && v) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: values go to a cache only", what);
  RotaryArgs a = {};
  if (to_cache) {
    a.ck = cache_part(cache_k, k_scale, strides, strides + 6);
    a.cv = cache_part(cache_v, v_scale, strides + 3, strides + 9);
    if (const int e = check_cache(what, a.ck, a.cv, n_pages, kv_heads, page, dim, kind)) return e;
    a.slots = slots, a.slots64 = slots64, a.page_shift = page_shift_of(page), a.n_slots = (long)n_pages * page;
  }
  if (tokens == 0 || (heads == 0 && kv_heads == 0)) return TRITEIA_HIP_OK;
  if ((heads && (!q || !q_out)) || (kv_heads && !k) || (to_cache ? !v || !slots || k_out : kv_heads && !k_out)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(table) || !aligned16(q_norm) || !aligned16(k_norm) ||
      !strides_ok({q_token, q_head, k_token, k_head, v_token, v_head}, 2, 16))
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: rows, table and norms need 16-byte alignment", what);
  a.q = q, a.k = k, a.v = v, a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
  a.q_out = q_out, a.k_out = k_out, a.tokens = tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.rot = rot;
  a.positions = positions, a.positions64 = positions64, a.table = static_cast<const float*>(table), a.limit = limit;
  a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps, a.inv_dim = 1.f / dim;
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  by_types(bf16, to_cache ? kind : kCacheSame, RotaryLaunch{a, interleaved, static_cast<hipStream_t>(stream)});
  return check_launch("rotary_cache_kernel");
}

int triteia_hip_cache_read(const void* cache_k, const void* cache_v, const void* k_scale, const void* v_scale, const long* strides, int n_pages, int kv_heads,
                           int page, int dim, int kind, const void* slots, int slots64, int tokens, void* k_out, void* v_out, int bf16, int dev, void* stream) {
  const char* what = "cache_read";
  if (!strides) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null strides", what);
  if (dim < 8 || dim > 256 || dim % 8 != 0) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: heads of %d elements: a multiple of 8 up to 256", what, dim);
  CacheReadArgs a = {};
  a.ck = cache_part(cache_k, k_scale, strides, strides + 6);
  a.cv = cache_part(cache_v, v_scale, strides + 3, strides + 9);
  if (const int e = check_cache(what, a.ck, a.cv, n_pages, kv_heads, page, dim, kind)) return e;
  if (tokens < 0 || (long)tokens * kv_heads > (1L << 31)) return fail(TRITEIA_HIP_ERR_PROB_SHAPE, "%s: %d tokens of %d heads", what, tokens, kv_heads);
  if (tokens == 0) return TRITEIA_HIP_OK;
  if (!slots || !k_out || !v_out) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: outputs need 16-byte alignment", what);
  a.k_out = k_out, a.v_out = v_out, a.slots = slots, a.slots64 = slots64, a.tokens = tokens, a.kv_heads = kv_heads, a.dim = dim;
  a.page_shift = page_shift_of(page), a.n_slots = (long)n_pages * page;
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  by_types(bf16, kind, ReadLaunch{a, static_cast<hipStream_t>(stream)});
  return check_launch("cache_read_kernel");
}

size_t triteia_hip_attention_plan_bytes(int n_seqs, int n_tokens, int heads, int kv_heads, int max_q) {
  if (check_batch("attention_plan", n_seqs, n_tokens, heads, kv_heads, max_q, 1, 0)) return 0;
  return 4 * (size_t)attn_layout(n_seqs, n_tokens, heads, kv_heads, max_q, 1, 0).ints;
}

size_t triteia_hip_attention_scratch_bytes(int n_seqs, int n_tokens, int heads, int kv_heads, int max_q, int dim) {
  if (check_batch("paged_attention", n_seqs, n_tokens, heads, kv_heads, max_q, 1, 0)) return 0;
  const AttnLayout l = attn_layout(n_seqs, n_tokens, heads, kv_heads, max_q, 1, 0);
  size_t bytes = 0;
  for (const AttnList& x : l.list) bytes += 4 * (size_t)x.max_parts * kv_heads * x.rows * (dim + 2);
  return bytes;
}

int triteia_hip_attention_plan(const void* q_starts, const void* kv_lens, int n_seqs, int n_tokens, int heads, int kv_heads, int max_q, int causal, int window,
                               void* plan, size_t plan_bytes, int dev, void* stream) {
  if (const int e = check_batch("attention_plan", n_seqs, n_tokens, heads, kv_heads, max_q, causal, window)) return e;
  if (n_tokens == 0) return TRITEIA_HIP_OK;
  const AttnLayout l = attn_layout(n_seqs, n_tokens, heads, kv_heads, max_q, causal, window);
  if (!q_starts || (n_seqs && !kv_lens) || !plan) return fail(TRITEIA_HIP_ERR_ARGUMENT, "attention_plan: null tensor pointer");
  if (plan_bytes < 4 * (size_t)l.ints || !aligned16(plan))
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "attention_plan: a plan of %zu bytes, 16-byte aligned, is needed, got %zu", 4 * (size_t)l.ints, plan_bytes);
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  hipLaunchKernelGGL(attention_plan_kernel, dim3(1), dim3(kAttnPlanThreads), 0, static_cast<hipStream_t>(stream), static_cast<const int*>(q_starts),
                     static_cast<const int*>(kv_lens), l, static_cast<int*>(plan));
  return check_launch("attention_plan_kernel");
}

int triteia_hip_paged_attention(const void* q, long q_token, long q_head, void* out, const void* cache_k, const void* cache_v, const void* k_scale, const void* v_scale,
                                const long* strides, int n_pages, int page, int kind, const void* pages, long pages_seq, int table_width, const void* plan,
                                size_t plan_bytes, int n_seqs, int n_tokens, int heads, int kv_heads, int dim, int max_q, int causal, int window, float scale,
                                void* scratch, size_t scratch_bytes, int bf16, int dev, void* stream) {
  const char* what = "paged_attention";
  if (const int e = check_batch(what, n_seqs, n_tokens, heads, kv_heads, max_q, causal, window)) return e;
  if (dim != 64 && dim != 128) return fail(TRITEIA_HIP_ERR_KERN_SHAPE, "%s: heads of %d elements: 64 or 128", what, dim);
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a scale of %g: a positive number", what, (double)scale);
  if (!strides) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null strides", what);
  AttendArgs a = {};
  a.ck = cache_part(cache_k, k_scale, strides, strides + 6);
  a.cv = cache_part(cache_v, v_scale, strides + 3, strides + 9);
  if (const int e = check_cache(what, a.ck, a.cv, n_pages, kv_heads, page, dim, kind)) return e;
  const long size = kind == kCacheSame ? 2 : 1;
  for (const CachePart* p : {&a.ck, &a.cv}) {
    if (!strides_ok({p->page, p->head, p->slot}, size, 16)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a cache's rows need 16-byte alignment", what);
    if (p->slot * size > (1L << 25)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: rows of a page %ld elements apart are too far", what, p->slot);
    if (kind != kCacheSame && (!aligned16(p->scale) || p->scale_slot != 1 || !strides_ok({p->scale_page, p->scale_head}, 4, 16)))
      return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a page's scales of one head have to be adjacent and 16-byte aligned", what);
  }
  if (n_tokens == 0) return TRITEIA_HIP_OK;
  const AttnLayout l = attn_layout(n_seqs, n_tokens, heads, kv_heads, max_q, causal, window);
  if (n_seqs > 0 && (table_width < 1 || !pages)) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: a table of pages with a column at least", what);
  if (!q || !out || !plan || !scratch) return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: null tensor pointer", what);
  if (!aligned16(q) || !aligned16(out) || !aligned16(plan) || !aligned16(scratch) || !strides_ok({q_token, q_head}, 2, 16))
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: queries, output, plan and scratch need 16-byte alignment", what);
  if (plan_bytes < 4 * (size_t)l.ints || scratch_bytes < triteia_hip_attention_scratch_bytes(n_seqs, n_tokens, heads, kv_heads, max_q, dim))
    return fail(TRITEIA_HIP_ERR_ARGUMENT, "%s: plan or scratch too small", what);
  a.q = q, a.q_token = q_token, a.q_head = q_head, a.out = out;
  a.pages = static_cast<const int*>(pages), a.pages_seq = pages_seq, a.n_pages = n_pages, a.table_width = table_width, a.page_shift = page_shift_of(page);
  a.held = (long)table_width * page < kAttnMaxTokens ? table_width * page : kAttnMaxTokens;
  a.group = heads / kv_heads, a.kv_heads = kv_heads, a.causal = causal, a.window = window, a.scale_log2 = scale * 1.44269504088896340736f;
  a.plan = static_cast<const int*>(plan);
  DeviceGuard g(dev);
  if (!g.ok) return fail(TRITEIA_HIP_ERR_RUNTIME, "cannot select device %d", dev);
  by_types(bf16, kind, AttendLaunch{a, l, static_cast<float*>(scratch), (long)table_width * page, dim, static_cast<hipStream_t>(stream)});
  return check_launch("paged attention");
}

}  // extern "C"
