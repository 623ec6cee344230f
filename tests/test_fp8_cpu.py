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
    (dict(x_type=2), ARGUMENT), (dict(x_type=2, xs=ONE, xs_token=-1), ARGUMENT), (dict(stride=12), ARGUMENT), (dict(w_stride=24), ARGUMENT), (dict(w_stride=(1 << 24) + 16), ARGUMENT), (dict(w=ODD), ARGUMENT),
    (dict(ws_row=-2), ARGUMENT), (dict(tokens=40, scratch=NULL), ARGUMENT), (dict(tokens=40, scratch=ODD), ARGUMENT), (dict(tokens=40, scratch_bytes=64), ARGUMENT)])
def test_product_refusals(what, code):
    assert matmul(**what) == code
    assert code == 0 or _ffi.last_error() != ""


def test_sizes_of_scratch():
    need = _ffi.lib().triteia_hip_fp8_scratch_bytes
    assert need(0, 8, 256, 0) == need(4, 0, 256, 0) == need(4, 8, 24, 0) == need(-1, 8, 256, 0) == need(4, 8, 0, 0) == 0
    for tokens in (1, 7, 16, 100, 5000):
        for m, k in ((1, 16), (1001, 2000), (4096, 4096), (28672, 8192)):
            codes = tokens * (k + 4 * -(-k // 128))
            assert need(tokens, m, k, 0) == need(tokens, m, k, 1) and need(tokens, m, k, 2) <= need(tokens, m, k, 0)
            assert tokens <= 4 or need(tokens, m, k, 2) <= need(tokens, m, k, 0) - codes          # (few tokens may be quantised on the way)
    assert need(1, 4096, 4096, 0) == need(4, 4096, 4096, 1) == 0 < need(5, 4096, 4096, 0)


def test_tiles():
    """Every tile has sizes that it is taken for; tests of the product run on all of them."""
    tile = _ffi.lib().triteia_hip_fp8_tile
    assert tile(0, 8, 256) == tile(1, 0, 256) == tile(1, 8, 24) == 0
    found = {tile(t, m, k) % 10 ** 6 for t in (1, 16, 17, 33, 48, 64, 100, 200, 300, 700, 1000, 2000, 8000) for m in (16, 640, 1001, 2050, 4096, 11008, 28672)
             for k in (128, 1040, 2000, 4096, 8192, 11008)}
    assert found >= {16016, 32016, 32032, 128016, 128032, 64064, 128064, 128096, 128128, 128160, 256096, 256128, 256192, 256224, 256256}, found
    assert tile(1, 4096, 4096) == 1016016 and tile(8000, 28672, 8192) == 1256256 and tile(64, 28672, 8192) == 1128064
    assert tile(128, 4096, 11008) // 10 ** 6 > 1                                # a long K over few tiles: in shares


def test_wait_states_ahead_of_direct_loads(tmp_path):
    """As of the other kernels: a scalar write of M0 is never right ahead of the load that uses it, of 16 bytes or 4, and a scalar base written by the vector unit five."""
    import re

    from tests.test_direct_loads_cpu import _kernels
    seen = set()
    for kernel, code in _kernels(tmp_path).items():
        for i, instruction in enumerate(code):
            if "fp8_" not in kernel or not instruction.startswith("global_load_lds"):
                continue
            seen.add((re.search(r"fp8_(tile|stream)", kernel).group(1), instruction.split()[0]))
            before = code[max(0, i - 5):i]
            assert not re.match(r"\S+ m0\b", before[-1]), (kernel, before[-1], instruction)
            scalars = re.search(r"s\[(\d+):(\d+)\]", instruction)
            if scalars:
                assert not [b for b in before if re.match(rf"v_\S+ s(\[?)({scalars.group(1)}|{scalars.group(2)})\b", b)], (kernel, before, instruction)
    assert seen == {(kind, "global_load_lds_" + size) for kind in ("tile", "stream") for size in ("dwordx4", "dword")}


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


def test_layer_keeps_the_types_of_its_base():
    """Conversions of a whole model leave codes and scales what they are, and move them."""
    from triteia_amd.python.nn import multi_delta_attention
    model = torch.nn.Sequential(multi_delta_attention(256, 4, 2, 64, 1, with_base="fp8"))
    layer = model[0].qkv_proj
    layer.base_scale.fill_(0.1)
    layer.base.view(torch.uint8).fill_(0x31)
    for convert in (model.half, model.double, lambda: model.to(torch.bfloat16), lambda: model.to("cpu")):
        convert()
        assert layer.base.dtype == torch.float8_e4m3fn and bool((layer.base.view(torch.uint8) == 0x31).all())
        assert torch.equal(layer.base_scale, torch.full((4, 2), 0.1)) and set(layer.state_dict()) == {"qweight", "meta", "scale", "base", "base_scale"}
    assert layer.to("meta").base.dtype == torch.float8_e4m3fn and layer.base_scale.device.type == "meta"
    for with_base in (None, False, True, 1):
        from triteia_amd.python.nn import multi_delta_linear
        dense = multi_delta_linear(256, 256, 1, with_base=with_base)
        assert (dense.base is None) == (not with_base) and "base_scale" not in dense.state_dict()
