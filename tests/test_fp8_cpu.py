"""The product in 8 bits without a GPU: import paths, refusals of the C entry points ahead of any launch, the native calls' way back to Python."""
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
ODD = ctypes.c_void_p(8)


def test_import_paths():
    import triteia  # noqa: F401
    for name in ("capi.fp8", "ops.matmul.fp8"):
        assert importlib.import_module("triteia.python." + name) is importlib.import_module("triteia_amd.python." + name)
    for name in ("quantize_fp8", "dequantize_fp8", "matmul_fp8"):
        assert callable(getattr(ops, name))


def quantize(x=ONE, stride=256, n=4, k=256, rows=1, codes=ONE, codes_stride=256, scales=ONE, row=1, block=4):
    return _ffi.lib().triteia_hip_fp8_quantize(x, stride, n, k, rows, codes, codes_stride, scales, row, block, 0, 0, NULL)


def values(codes=ONE, stride=256, scales=ONE, row=1, block=4, rows=1, n=4, k=256, out=ONE, kind=0):
    return _ffi.lib().triteia_hip_fp8_values(codes, stride, scales, row, block, rows, n, k, out, kind, 0, NULL)


def matmul(x=ONE, stride=256, x_type=0, xs=NULL, xs_token=0, xs_block=0, w=ONE, w_stride=256, ws=ONE, ws_row=2, ws_block=1, out=ONE, kind=0, tokens=4, m=8, k=256,
           scratch=ONE, scratch_bytes=1 << 40):
    return _ffi.lib().triteia_hip_fp8_matmul(x, stride, x_type, xs, xs_token, xs_block, w, w_stride, ws, ws_row, ws_block, out, kind, tokens, m, k, scratch,
                                             scratch_bytes, 0, NULL)


SHAPE, KERNEL, ARGUMENT = _ffi.ERR_PROB_SHAPE, _ffi.ERR_KERN_SHAPE, _ffi.ERR_ARGUMENT


@pytest.mark.parametrize("what,code", [
    (dict(n=0), 0), (dict(k=0), 0), (dict(n=-1), SHAPE), (dict(k=-16), SHAPE), (dict(k=24), SHAPE), (dict(n=(1 << 24) + 1), SHAPE), (dict(rows=2), KERNEL), (dict(rows=0), KERNEL),
    (dict(x=NULL), ARGUMENT), (dict(codes=NULL), ARGUMENT), (dict(scales=NULL), ARGUMENT), (dict(x=ODD), ARGUMENT), (dict(stride=4), ARGUMENT), (dict(stride=-8), ARGUMENT),
    (dict(codes_stride=252), ARGUMENT), (dict(codes_stride=128), ARGUMENT), (dict(row=-1), ARGUMENT), (dict(block=-1), ARGUMENT), (dict(scales=ctypes.c_void_p(2)), ARGUMENT),
    (dict(n=1 << 24, k=1 << 20, codes_stride=1 << 20), SHAPE)])
def test_quantiser_refusals(what, code):
    assert quantize(**what) == code
    assert code == 0 or _ffi.last_error() != ""


@pytest.mark.parametrize("what,code", [
    (dict(n=0), 0), (dict(k=24), SHAPE), (dict(rows=3), KERNEL), (dict(kind=3), KERNEL), (dict(kind=-1), KERNEL), (dict(codes=NULL), ARGUMENT), (dict(out=NULL), ARGUMENT),
    (dict(out=ODD), ARGUMENT), (dict(stride=12), ARGUMENT), (dict(scales=NULL), ARGUMENT), (dict(row=-1), ARGUMENT)])
def test_read_back_refusals(what, code):
    assert values(**what) == code
    assert code == 0 or _ffi.last_error() != ""


@pytest.mark.parametrize("what,code", [
    (dict(tokens=0), 0), (dict(m=0), 0), (dict(k=0), SHAPE), (dict(k=24), SHAPE), (dict(tokens=-1), SHAPE), (dict(m=-1), SHAPE), (dict(m=(1 << 24) + 1), SHAPE),
    (dict(x_type=3), KERNEL), (dict(kind=3), KERNEL), (dict(x=NULL), ARGUMENT), (dict(w=NULL), ARGUMENT), (dict(ws=NULL), ARGUMENT), (dict(out=NULL), ARGUMENT),
    (dict(x_type=2), ARGUMENT), (dict(x_type=2, xs=ONE, xs_token=-1), ARGUMENT), (dict(stride=12), ARGUMENT), (dict(w_stride=24), ARGUMENT), (dict(w=ODD), ARGUMENT),
    (dict(ws_row=-2), ARGUMENT), (dict(scratch=NULL), ARGUMENT), (dict(scratch=ODD), ARGUMENT), (dict(scratch_bytes=64), ARGUMENT)])
def test_product_refusals(what, code):
    assert matmul(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def test_sizes_of_scratch():
    need = _ffi.lib().triteia_hip_fp8_scratch_bytes
    assert need(0, 8, 256, 0) == need(4, 0, 256, 0) == need(4, 8, 24, 0) == need(-1, 8, 256, 0) == need(4, 8, 0, 0) == 0
    for tokens in (1, 7, 16, 100, 5000):
        for m, k in ((1, 16), (1001, 2000), (4096, 4096), (28672, 8192)):
            codes = tokens * (k + 4 * -(-k // 128))
            assert codes <= need(tokens, m, k, 0) == need(tokens, m, k, 1) and need(tokens, m, k, 2) <= need(tokens, m, k, 0) - codes


class Subclass(torch.Tensor):
    """Any subclass: it may give every operation another meaning."""


FUNCTIONS = {"quantize_fp8": 2, "dequantize_fp8": 3, "matmul_fp8": 5}


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
    x = torch.zeros(3, 256, dtype=torch.float16)
    codes, scales = x.to(torch.float8_e4m3fn), torch.ones(3, 2)
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.dequantize_fp8(codes, scales), lambda: ops.matmul_fp8(x, codes, torch.ones(1, 2))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
