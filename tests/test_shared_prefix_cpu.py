"""Attention over shared prefixes without a GPU: refusals of the C entry points ahead of any launch, sizes, the native calls' way back to Python."""
import ctypes

import numpy as np
import pytest
import torch

from triteia_amd.python import ops
from triteia_amd.python.capi import _ffi
from triteia_amd.python.capi._native import native

NULL = ctypes.c_void_p(0)
ONE = ctypes.c_void_p(16)          # (an aligned address that no refused call follows)
STRIDES = (ctypes.c_long * 12)(4096, 2048, 128, 4096, 2048, 128, 32, 16, 1, 32, 16, 1)


def plan(seqs=4, groups=2, tokens=4, heads=4, kv_heads=2, max_q=1, causal=1, window=0, starts=ONE, lens=ONE, group_starts=ONE, prefixes=ONE, out=ONE, nbytes=1 << 30):
    return _ffi.lib().triteia_hip_shared_plan(starts, lens, group_starts, prefixes, seqs, groups, tokens, heads, kv_heads, max_q, causal, window, out, nbytes, 0, NULL)


@pytest.mark.parametrize("what,code", [
    (dict(tokens=0), 0), (dict(groups=-1), _ffi.ERR_PROB_SHAPE), (dict(groups=1025), _ffi.ERR_PROB_SHAPE), (dict(seqs=4000, groups=97), _ffi.ERR_PROB_SHAPE),
    (dict(seqs=-1), _ffi.ERR_PROB_SHAPE), (dict(heads=3), _ffi.ERR_PROB_SHAPE), (dict(causal=0, window=3), _ffi.ERR_ARGUMENT), (dict(starts=NULL), _ffi.ERR_ARGUMENT),
    (dict(lens=NULL), _ffi.ERR_ARGUMENT), (dict(group_starts=NULL), _ffi.ERR_ARGUMENT), (dict(prefixes=NULL), _ffi.ERR_ARGUMENT), (dict(out=NULL), _ffi.ERR_ARGUMENT),
    (dict(out=ctypes.c_void_p(8)), _ffi.ERR_ARGUMENT), (dict(nbytes=64), _ffi.ERR_ARGUMENT)])
def test_plan_refusals(what, code):
    assert plan(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def attend(seqs=4, groups=2, tokens=4, heads=4, kv_heads=2, dim=128, scale=0.1, plan_bytes=1 << 30, scratch_bytes=1 << 34, strides=STRIDES, width=2):
    return _ffi.lib().triteia_hip_shared_attention(ONE, 512, 128, ONE, ONE, ONE, ONE, ONE, strides, 2, 16, 0, ONE, 2, width, ONE, plan_bytes, seqs, groups, tokens, heads, kv_heads,
                                                   dim, 1, 1, 0, scale, ONE, scratch_bytes, 0, 0, NULL)


@pytest.mark.parametrize("what,code", [
    (dict(tokens=0), 0), (dict(groups=1025), _ffi.ERR_PROB_SHAPE), (dict(groups=-1), _ffi.ERR_PROB_SHAPE), (dict(seqs=4096), _ffi.ERR_PROB_SHAPE), (dict(dim=96), _ffi.ERR_KERN_SHAPE),
    (dict(scale=0.0), _ffi.ERR_ARGUMENT), (dict(plan_bytes=16), _ffi.ERR_ARGUMENT), (dict(scratch_bytes=16), _ffi.ERR_ARGUMENT), (dict(strides=None), _ffi.ERR_ARGUMENT),
    (dict(width=0), _ffi.ERR_ARGUMENT)])
def test_attention_refusals(what, code):
    assert attend(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def test_sizes():
    """Without groups the sizes of the ordinary plan, with them never less than with fewer, and enough for a result of every row in shares of its own and of the prefix."""
    lib = _ffi.lib()
    for heads, kv_heads in ((32, 32), (64, 8), (20, 1), (3, 3)):
        for seqs, tokens, max_q in ((1, 1, 1), (2, 2, 1), (8, 50, 30), (64, 64, 1), (512, 4000, 100)):
            sizes = (tokens, heads, kv_heads, max_q)
            assert lib.triteia_hip_shared_plan_bytes(seqs, 0, *sizes) == lib.triteia_hip_attention_plan_bytes(seqs, *sizes)
            assert lib.triteia_hip_shared_scratch_bytes(seqs, 0, *sizes, 64) == lib.triteia_hip_attention_scratch_bytes(seqs, *sizes, 64)
            held = [lib.triteia_hip_shared_scratch_bytes(seqs, groups, *sizes, 64) for groups in (1, 2, 5, 30)]
            assert all(0 < a <= b for a, b in zip(held, held[1:])) and (seqs == 1 or held[0] >= 2 * tokens * heads * 66 * 4)
    assert lib.triteia_hip_shared_plan_bytes(4, 1025, 4, 4, 2, 1) == 0 and lib.triteia_hip_shared_scratch_bytes(4, 1025, 4, 4, 2, 1, 64) == 0


@pytest.mark.parametrize("heads,kv_heads", [(64, 8), (32, 32), (32, 4), (20, 1)])
@pytest.mark.parametrize("seqs,groups", [(1, 1), (8, 1), (16, 3), (64, 1), (200, 20)])
def test_scratch_of_prompts(heads, kv_heads, seqs, groups):
    """Prompts share nothing, and no number of their tokens takes more: beside the scratch without groups there is that of the rows that may share, 64 a sequence and 6144, in tiles of 128, and of
    the tiles that a sequence or a group leaves part empty, each for the rows themselves and for the prefix."""
    lib, dim, group = _ffi.lib(), 128, heads // kv_heads
    rows = 64 * seqs + 6144
    tiles = 2 * rows // 128 + 2 * (seqs + groups + 1)
    allowed = 4 * kv_heads * (dim + 2) * (128 * tiles + 48 * (seqs + groups + 1)) + 2 * 1024 * 32 * (dim + 2) * 4
    for max_q in (1, 4096):
        sizes = []
        for tokens in (8192, 32768, 131072, 1 << 20):
            held = lib.triteia_hip_shared_scratch_bytes(seqs, groups, tokens, heads, kv_heads, max_q, dim)
            alone = lib.triteia_hip_attention_scratch_bytes(seqs, tokens, heads, kv_heads, 4096, dim)
            assert 0 < held <= alone + allowed, (tokens, held, alone, allowed)
            if group * tokens >= rows + 128 * seqs:
                sizes.append(held)
        assert max(sizes) <= 1.02 * min(sizes), sizes
    eight = lib.triteia_hip_shared_scratch_bytes(8, 1, 131072, 64, 8, 131072, 128), lib.triteia_hip_attention_scratch_bytes(8, 131072, 64, 8, 131072, 128)
    assert eight[0] <= 1.2 * eight[1], eight


class Subclass(torch.Tensor):
    """Any subclass: it may give every operation another meaning."""


@pytest.mark.parametrize("name,n", [("shared_plan", 10), ("shared_attention", 14)])
def test_native_calls_leave_what_is_not_plain(name, n):
    fn = getattr(native(), name)
    for strange in (None, [0, 1], np.zeros(3, dtype=np.int32), 3, 1.5, True, "x", torch.float16, object(), torch.zeros(2, 2), torch.zeros(2, 2).as_subclass(Subclass), 1 << 80):
        assert fn(*[strange] * n) is None
        for i in range(n):
            assert fn(*[torch.zeros(2, 2)] * i, strange, *[torch.zeros(2, 2)] * (n - i - 1)) is None
    for count in (0, 1, n - 1, n + 1, 40):
        assert fn(*[torch.zeros(2, 2)] * count) is None


def test_ops_refuse_the_cpu():
    class Cache:
        kv_heads = 2
    whole = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.attention_plan(Cache, whole, whole[:2], 4, 2, group_starts=whole[:2], prefix_lens=whole[:1])
