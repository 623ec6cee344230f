"""Entry points of the attention side of a serving step: rotary positions, the paged cache and the attention over it.  The reference
has no counterpart."""
import ctypes

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _ffi
from ._native import native

_DTYPES = (torch.float16, torch.bfloat16)
_NONE = (None,) * 4
CACHE_KINDS = {torch.float16: 0, torch.bfloat16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}


def _check(err):
    if err == _ffi.ERR_RUNTIME:
        raise RuntimeError(f"triteia_hip error {err}: {_ffi.last_error()}")
    if err:
        raise RuntimeError(_ffi.last_error())


def _require(like=None, optional=(), **tensors):
    """GPU tensors of one device, in any layout, that record no gradient in either direction; those named in `optional` may be None."""
    for name, t in tensors.items():
        if t is None and name in optional:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a GPU tensor (this op has no CPU implementation)")
        if like is not None and t.device != like:
            raise RuntimeError(f"{name} is on {t.device}, expected {like}")
        like = t.device
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, which this op does not record")
        if unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has a tangent, which this op does not carry on")
    return like


def _rows(name, t, heads=None, dim=None):
    """A [tokens, heads, dim] tensor whose rows can be read 16 bytes at a time: `t` itself, or a copy."""
    if t.dim() != 3 or t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be [tokens, heads, dim] in torch.float16 or torch.bfloat16, got {tuple(t.shape)} in {t.dtype}")
    if (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected [tokens, {heads if heads is not None else t.shape[1]}, {dim}]")
    if t.is_neg() or (t.numel() and (t.stride(2) != 1 or any(s % 8 or s < 0 for s in t.stride()[:2]) or t.data_ptr() % 16)):
        return t.resolve_neg().clone(memory_format=torch.contiguous_format)
    return t


def _integers(name, t, n=None):
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name} must be torch.int32 or torch.int64, got {t.dtype}")
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise RuntimeError(f"{name} must have one entry for each of {n} tokens, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


class PagedCache:
    """Keys and values in pages: `k` and `v` [n_pages, kv_heads, page, dim] in fp16, bf16, int8 or float8_e4m3fn, the 8-bit types with
    `k_scale` and `v_scale` float32 [n_pages, kv_heads, page] (value = code * scale).  Views are fine as long as a row's elements are adjacent
    and rows start on 16 bytes (a head of fewer elements than that in 8 bits: 8), e.g. of tensors [n_pages, page, kv_heads, dim].

    Slot `page * (tokens of a page) + offset` names a token's place."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        device = _require(optional=("k_scale", "v_scale"), k=k, v=v, k_scale=k_scale, v_scale=v_scale)
        if k.dtype not in CACHE_KINDS or v.dtype != k.dtype:
            raise RuntimeError(f"a cache holds fp16, bf16, int8 or float8_e4m3fn, the same for k and v, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or v.shape != k.shape:
            raise RuntimeError(f"k and v must be [n_pages, kv_heads, page, dim], got {tuple(k.shape)} and {tuple(v.shape)}")
        n_pages, kv_heads, page, dim = k.shape
        if n_pages < 1 or kv_heads < 1 or page not in (16, 32, 64, 128, 256, 512, 1024):
            raise RuntimeError(f"a cache needs pages of 16, 32, .. 1024 tokens, one page and one head at least, got {tuple(k.shape)}")
        if n_pages * page > 2 ** 31 - 1:
            raise RuntimeError(f"a cache of {n_pages} pages of {page} tokens has more than 2^31 slots")
        if any(t is not None and t.is_neg() for t in (k, v, k_scale, v_scale)):
            raise RuntimeError("a cache of lazily negated tensors: its memory holds the other sign")
        kind = CACHE_KINDS[k.dtype]
        align = 16 // k.element_size() if kind == 0 or dim % 16 == 0 else 8
        for name, t in (("k", k), ("v", v)):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(s < 0 or s % align for s in t.stride()[:3]):
                raise RuntimeError(f"{name}'s rows must be of adjacent elements and start on whole {align * t.element_size()} bytes, got strides {t.stride()}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is None) != (kind == 0):
                raise RuntimeError(f"{name} belongs to caches of 8 bits")
            if t is not None and (t.dtype != torch.float32 or t.shape != k.shape[:3] or t.stride(2) != 1 or t.data_ptr() % 16
                                  or any(s < 0 or s % 4 for s in t.stride()[:2])):
                raise RuntimeError(f"{name} must be float32 {tuple(k.shape[:3])}, a page's scales of one head adjacent, got {t.dtype} {tuple(t.shape)} with "
                                   f"strides {t.stride()}")
        self._tensors = (k, v, k_scale, v_scale)
        self.n_pages, self.kv_heads, self.page, self.dim, self.kind, self.device, self.dtype = n_pages, kv_heads, page, dim, kind, device, k.dtype
        scales = [0] * 6 if kind == 0 else [*k_scale.stride(), *v_scale.stride()]
        self._strides = (ctypes.c_long * 12)(*k.stride()[:3], *v.stride()[:3], *scales)

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    def _pointers(self):
        return [_ffi.ptr(t) for t in self._tensors]

    def _activations(self, dtype):
        if dtype not in _DTYPES or (self.kind == 0 and dtype != self.dtype):
            raise RuntimeError(f"a cache of {self.dtype} does not go with activations of {dtype}")


def rotary_cache(q, k, v, positions, table, cache, slots, interleaved=False, q_norm=None, k_norm=None, eps=1e-6):
    """The one launch behind ops.rotary, ops.rotary_cache_write and ops.cache_write: (q, k) of the outputs, None where there is none."""
    held = cache._tensors if cache is not None else _NONE
    out = native().rotary_cache(q, k, v, positions, table, held[0], held[1], held[2], held[3], slots, interleaved, q_norm, k_norm, eps)
    if out is not None:
        return out
    if (positions is None) != (table is None):
        raise RuntimeError("positions and table go together")
    optional = ("q", "positions", "table", "q_norm", "k_norm") + (("v", "slots") if cache is None else ())
    device = _require(optional=optional, q=q, k=k, v=v, positions=positions, table=table, slots=slots, q_norm=q_norm, k_norm=k_norm)
    tokens, dim, dtype = k.shape[0], k.shape[-1], k.dtype
    if cache is not None:
        if cache.device != device:
            raise RuntimeError(f"the cache is on {cache.device}, expected {device}")
        cache._activations(dtype)
        v = _rows("v", v, cache.kv_heads, cache.dim)
        k = _rows("k", k, cache.kv_heads, cache.dim)
        slots = _integers("slots", slots, tokens)
    else:
        k = _rows("k", k, None, dim)
    if q is not None:
        q = _rows("q", q, None, dim)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t is not None and (t.shape[0] != tokens or t.dtype != dtype):
            raise RuntimeError(f"{name} is {tuple(t.shape)} in {t.dtype}, expected {tokens} tokens in {dtype}")
    if dim % 8 or not 8 <= dim <= 256:
        raise RuntimeError(f"heads of {dim} elements: a multiple of 8 up to 256")
    rot = limit = 0
    if positions is not None:
        positions = _integers("positions", positions, tokens)
        if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
            raise RuntimeError(f"table must be contiguous float32 [positions, pairs, 2], got {table.dtype} {tuple(table.shape)}")
        table = table.resolve_neg()
        limit, rot = table.shape[0], 2 * table.shape[1]
        if rot % 16 or not 16 <= rot <= dim or limit < 1:
            raise RuntimeError(f"a table of {limit} positions that rotates {rot} of {dim} elements: a position at least, a multiple of 16 elements")
    norms = []
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None and (t.shape != (dim,) or t.dtype != dtype):
            raise RuntimeError(f"{name} must be [{dim}] in {dtype}, got {tuple(t.shape)} in {t.dtype}")
        norms.append(t if t is None or (t.is_contiguous() and not t.is_neg() and t.data_ptr() % 16 == 0) else t.resolve_neg().clone(memory_format=torch.contiguous_format))
    q_out = torch.empty((tokens, q.shape[1], dim), dtype=dtype, device=device) if q is not None else None
    k_out = torch.empty((tokens, k.shape[1], dim), dtype=dtype, device=device) if cache is None else None
    strides = [s for t in (q, k, v) for s in (t.stride()[:2] if t is not None else (0, 0))]
    place = (*cache._pointers(), cache._strides, cache.n_pages, cache.page, cache.kind) if cache is not None else (None, None, None, None, None, 0, 0, 0)
    _check(_ffi.lib().triteia_hip_rotary_cache(
        _ffi.ptr(q), strides[0], strides[1], _ffi.ptr(k), strides[2], strides[3], _ffi.ptr(v), strides[4], strides[5], _ffi.ptr(q_out), _ffi.ptr(k_out),
        tokens, q.shape[1] if q is not None else 0, k.shape[1], dim, rot, _ffi.ptr(positions),
        int(positions is not None and positions.dtype == torch.int64), _ffi.ptr(table) if positions is not None else None, limit, int(bool(interleaved)),
        _ffi.ptr(norms[0]), _ffi.ptr(norms[1]), float(eps), _ffi.ptr(slots), int(slots is not None and slots.dtype == torch.int64), *place,
        int(dtype == torch.bfloat16), _ffi.device_index(k), _ffi.stream_of(k)))
    return q_out, k_out


def cache_read(cache, slots, dtype):
    """(k, v) [len(slots), kv_heads, dim] of the cache's rows at `slots`; zeros where a slot lies outside the cache."""
    out = native().cache_read(*cache._tensors, slots, dtype)
    if out is not None:
        return out
    _require(cache.device, slots=slots)
    cache._activations(dtype)
    slots = _integers("slots", slots, slots.shape[0] if slots.dim() else None)
    k, v = (torch.empty((slots.shape[0], cache.kv_heads, cache.dim), dtype=dtype, device=cache.device) for _ in range(2))
    _check(_ffi.lib().triteia_hip_cache_read(
        *cache._pointers(), cache._strides, cache.n_pages, cache.kv_heads, cache.page, cache.dim, cache.kind, _ffi.ptr(slots), int(slots.dtype == torch.int64),
        slots.shape[0], _ffi.ptr(k), _ffi.ptr(v), int(dtype == torch.bfloat16), _ffi.device_index(slots), _ffi.stream_of(slots)))
    return k, v


class AttentionPlan:
    """The work list of a batch (from `attention_plan`), for every layer of a forward pass whose heads are as many."""

    def __init__(self, buffer, n_seqs, n_tokens, heads, kv_heads, max_q, causal, window):
        self.buffer = buffer
        self.n_seqs, self.n_tokens, self.heads, self.kv_heads, self.max_q, self.causal, self.window = n_seqs, n_tokens, heads, kv_heads, max_q, causal, window


def attention_plan(q_starts, kv_lens, n_tokens, heads, kv_heads, max_q=None, causal=True, window=0):
    max_q = n_tokens if max_q is None else max_q
    buffer = native().attention_plan(q_starts, kv_lens, n_tokens, heads, kv_heads, max_q, causal, window)
    if buffer is not None:
        return AttentionPlan(buffer, kv_lens.shape[0], n_tokens, heads, kv_heads, max_q, bool(causal), window)
    device = _require(q_starts=q_starts, kv_lens=kv_lens)
    for name, t in (("q_starts", q_starts), ("kv_lens", kv_lens)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous vector of torch.int32, got {tuple(t.shape)} of {t.dtype}")
    n_seqs = kv_lens.shape[0]
    if q_starts.shape[0] != n_seqs + 1:
        raise RuntimeError(f"q_starts must have {n_seqs + 1} entries for {n_seqs} sequences, got {q_starts.shape[0]}")
    sizes = (n_seqs, int(n_tokens), int(heads), int(kv_heads), int(max_q))
    nbytes = _ffi.lib().triteia_hip_attention_plan_bytes(*sizes)
    if nbytes == 0:
        raise RuntimeError(_ffi.last_error())
    buffer = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _check(_ffi.lib().triteia_hip_attention_plan(_ffi.ptr(q_starts), _ffi.ptr(kv_lens), *sizes, int(bool(causal)), int(window), _ffi.ptr(buffer), nbytes,
                                                 _ffi.device_index(q_starts), _ffi.stream_of(q_starts)))
    return AttentionPlan(buffer, *sizes, bool(causal), int(window))


def paged_attention(q, cache, pages, plan, scale):
    if isinstance(q, torch.Tensor) and q.dim() == 3 and q.shape[0] == plan.n_tokens and cache.kv_heads == plan.kv_heads:
        out = native().paged_attention(q, *cache._tensors, pages, plan.buffer, plan.n_seqs, plan.heads, plan.max_q, plan.causal, plan.window, scale)
        if out is not None:
            return out
    device = _require(cache.device, q=q, pages=pages, plan=plan.buffer)
    cache._activations(q.dtype)
    q = _rows("q", q, plan.heads, cache.dim)
    if q.shape[0] != plan.n_tokens or cache.kv_heads != plan.kv_heads:
        raise RuntimeError(f"the plan is for {plan.n_tokens} tokens and {plan.kv_heads} heads of the cache, got {q.shape[0]} and {cache.kv_heads}")
    if pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[0] != plan.n_seqs or (pages.numel() and pages.stride(1) != 1) or (pages.numel() and pages.stride(0) < 0):
        raise RuntimeError(f"pages must be torch.int32 [{plan.n_seqs}, pages of a sequence], its rows adjacent, got {pages.dtype} {tuple(pages.shape)}")
    out = torch.empty((plan.n_tokens, plan.heads, cache.dim), dtype=q.dtype, device=device)
    sizes = (plan.n_seqs, plan.n_tokens, plan.heads, plan.kv_heads, plan.max_q)
    nbytes = _ffi.lib().triteia_hip_attention_scratch_bytes(*sizes, cache.dim)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _check(_ffi.lib().triteia_hip_paged_attention(
        _ffi.ptr(q), q.stride(0), q.stride(1), _ffi.ptr(out), *cache._pointers(), cache._strides, cache.n_pages, cache.page, cache.kind, _ffi.ptr(pages),
        pages.stride(0), pages.shape[1], _ffi.ptr(plan.buffer), plan.buffer.numel(), plan.n_seqs, plan.n_tokens, plan.heads, plan.kv_heads, cache.dim, plan.max_q,
        int(plan.causal), plan.window, float(scale), _ffi.ptr(scratch), nbytes, int(q.dtype == torch.bfloat16), _ffi.device_index(q), _ffi.stream_of(q)))
    return out
