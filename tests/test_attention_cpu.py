"""The attention side without a GPU: import paths, refusals of the C entry points ahead of any launch, the native calls' way back to Python."""
import ctypes
import importlib

import numpy as np
import pytest
import torch

from triteia_amd.python import ops
from triteia_amd.python.capi import _ffi
from triteia_amd.python.capi._native import native

NULL = ctypes.c_void_p(0)
ONE = ctypes.c_void_p(16)          # (an aligned address that no refused call follows)
STRIDES = (ctypes.c_long * 12)(4096, 2048, 128, 4096, 2048, 128, 32, 16, 1, 32, 16, 1)


def test_import_paths():
    import triteia  # noqa: F401
    for name in ("capi.attention", "ops.attention", "ops.attention.rotary", "ops.attention.cache", "ops.attention.paged", "nn.attention"):
        assert importlib.import_module("triteia.python." + name) is importlib.import_module("triteia_amd.python." + name)
    for name in ("rotary_table", "rotary", "rotary_cache_write", "PagedCache", "paged_cache", "cache_write", "cache_read", "attention_plan", "paged_attention"):
        assert callable(getattr(ops, name))


def rotary(tokens=4, heads=2, kv_heads=2, dim=128, rot=128, positions=ONE, table=ONE, limit=10, q=ONE, k_out=ONE, strides=None, v=NULL, page=16, kind=0, n_pages=2,
           slots=ONE, q_token=256):
    cache = NULL if strides is None else ONE
    return _ffi.lib().triteia_hip_rotary_cache(q, q_token, 128, ONE, 256, 128, v, 256, 128, ONE, k_out, tokens, heads, kv_heads, dim, rot, positions, 0, table, limit, 0, NULL,
                                               NULL, 1e-6, slots, 0, cache, cache, cache, cache, strides, n_pages, page, kind, 0, 0, NULL)


@pytest.mark.parametrize("what,code", [
    (dict(tokens=0), 0), (dict(tokens=-1), _ffi.ERR_PROB_SHAPE), (dict(dim=12), _ffi.ERR_KERN_SHAPE), (dict(dim=264), _ffi.ERR_KERN_SHAPE),
    (dict(rot=8), _ffi.ERR_KERN_SHAPE), (dict(rot=144), _ffi.ERR_KERN_SHAPE), (dict(table=NULL), _ffi.ERR_KERN_SHAPE), (dict(limit=0), _ffi.ERR_KERN_SHAPE),
    (dict(q=NULL), _ffi.ERR_ARGUMENT), (dict(q=ctypes.c_void_p(8)), _ffi.ERR_ARGUMENT), (dict(q_token=4), _ffi.ERR_ARGUMENT), (dict(k_out=NULL), _ffi.ERR_ARGUMENT),
    (dict(v=ONE), _ffi.ERR_ARGUMENT), (dict(strides=STRIDES, k_out=NULL), _ffi.ERR_ARGUMENT), (dict(strides=STRIDES, k_out=NULL, v=ONE, slots=NULL), _ffi.ERR_ARGUMENT),
    (dict(strides=STRIDES, k_out=NULL, v=ONE, page=24), _ffi.ERR_PROB_SHAPE), (dict(strides=STRIDES, k_out=NULL, v=ONE, kind=3), _ffi.ERR_KERN_SHAPE),
    (dict(strides=STRIDES, k_out=NULL, v=ONE, n_pages=0), _ffi.ERR_PROB_SHAPE)])
def test_rotary_refusals(what, code):
    assert rotary(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def attend(seqs=2, tokens=4, heads=4, kv_heads=2, dim=128, max_q=2, causal=1, window=0, scale=0.1, q=ONE, plan_bytes=1 << 30, scratch_bytes=1 << 34, width=2, strides=STRIDES):
    return _ffi.lib().triteia_hip_paged_attention(q, 512, 128, ONE, ONE, ONE, ONE, ONE, strides, 2, 16, 0, ONE, 2, width, ONE, plan_bytes, seqs, tokens, heads, kv_heads, dim, max_q,
                                                  causal, window, scale, ONE, scratch_bytes, 0, 0, NULL)


@pytest.mark.parametrize("what,code", [
    (dict(tokens=0), 0), (dict(seqs=4097), _ffi.ERR_PROB_SHAPE), (dict(heads=5), _ffi.ERR_PROB_SHAPE), (dict(kv_heads=0), _ffi.ERR_PROB_SHAPE),
    (dict(dim=96), _ffi.ERR_KERN_SHAPE), (dict(causal=0, window=3), _ffi.ERR_ARGUMENT), (dict(window=-1), _ffi.ERR_PROB_SHAPE), (dict(scale=0.0), _ffi.ERR_ARGUMENT),
    (dict(scale=float("nan")), _ffi.ERR_ARGUMENT), (dict(scale=float("inf")), _ffi.ERR_ARGUMENT), (dict(q=NULL), _ffi.ERR_ARGUMENT), (dict(q=ctypes.c_void_p(8)), _ffi.ERR_ARGUMENT),
    (dict(plan_bytes=16), _ffi.ERR_ARGUMENT), (dict(scratch_bytes=16), _ffi.ERR_ARGUMENT), (dict(width=0), _ffi.ERR_ARGUMENT), (dict(strides=None), _ffi.ERR_ARGUMENT)])
def test_attention_refusals(what, code):
    assert attend(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def test_sizes_of_plan_and_scratch():
    """What the host allocates covers any lengths of the batch: more tokens, sequences or new tokens of one never need less."""
    lib = _ffi.lib()
    assert lib.triteia_hip_attention_plan_bytes(5000, 10, 4, 2, 1) == 0 and lib.triteia_hip_attention_scratch_bytes(1, 10, 5, 2, 1, 128) == 0
    for heads, kv_heads in ((32, 32), (64, 8), (20, 1), (3, 3)):
        for max_q in (1, 2, 16, 1000):
            sizes = [lib.triteia_hip_attention_plan_bytes(seqs, tokens, heads, kv_heads, max_q) for seqs, tokens in ((1, 1), (1, 50), (8, 50), (64, 400), (512, 4000))]
            assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
            assert lib.triteia_hip_attention_scratch_bytes(8, 50, heads, kv_heads, max_q, 128) >= 0


class Subclass(torch.Tensor):
    """Any subclass: it may give every operation another meaning."""


FUNCTIONS = {"rotary_cache": 14, "cache_read": 6, "attention_plan": 8, "paged_attention": 13}


@pytest.mark.parametrize("name", sorted(FUNCTIONS))
def test_native_calls_leave_what_is_not_plain(name):
    fn, n = getattr(native(), name), FUNCTIONS[name]
    for strange in (None, [0, 1], np.zeros(3, dtype=np.int32), 3, 1.5, True, "x", torch.float16, object(), torch.zeros(2, 2), torch.zeros(2, 2).as_subclass(Subclass), 1 << 80):
        assert fn(*[strange] * n) is None
        for i in range(n):
            assert fn(*[torch.zeros(2, 2)] * i, strange, *[torch.zeros(2, 2)] * (n - i - 1)) is None
    for count in (0, 1, n - 1, n + 1, 40):
        assert fn(*[torch.zeros(2, 2)] * count) is None


def test_ops_refuse_the_cpu():
    x, table = torch.zeros(3, 2, 64, dtype=torch.float16), ops.rotary_table(10, 64, device="cpu")
    positions = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.rotary(x, x, positions, table)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.paged_cache(4, 2, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.PagedCache(torch.zeros(2, 2, 16, 64, dtype=torch.float16), torch.zeros(2, 2, 16, 64, dtype=torch.float16))
