"""Entry points of the base weight in 8 bits: the quantiser, its read-back and the product.  (The reference's FP8 layer, nn/linear.py:144-175, calls torch's product
with one scale for a whole tensor.)"""
import torch

from . import _ffi
from ._native import native
from .attention import _check, _require

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
BLOCK = 128


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _adjacent(t, rows):
    """Rows of adjacent elements that start on 16 bytes: `t` [rows, k] itself, or a copy."""
    t = t.reshape(rows, t.shape[-1])
    if t.is_neg() or (t.numel() and (t.stride(1) != 1 or not 0 <= t.stride(0) <= 1 << 24 or t.stride(0) * t.element_size() % 16 or t.data_ptr() % 16)):
        return t.resolve_neg().clone(memory_format=torch.contiguous_format)
    return t


def _scales(name, t, rows, k):
    if t.dtype != torch.float32 or t.shape != (rows, _blocks(k)):
        raise RuntimeError(f"{name} must be torch.float32 [{rows}, {_blocks(k)}], one for each block of {BLOCK}, got {t.dtype} {tuple(t.shape)}")
    return t.resolve_neg()


def _width(name, k):
    if k % 16 or k < 16:
        raise RuntimeError(f"{name} has rows of {k} elements: a multiple of 16")


def quantize_fp8(x, rows):
    out = native().quantize_fp8(x, rows)
    if out is not None:
        return out
    device = _require(x=x)
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        raise RuntimeError(f"x must be [rows, elements] in torch.float16 or torch.bfloat16, got {tuple(x.shape)} in {x.dtype}")
    if rows not in (1, BLOCK):
        raise RuntimeError(f"{rows} rows of a scale: 1 or {BLOCK}")
    n, k = x.shape
    _width("x", k)
    x = _adjacent(x, n)
    codes = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty((_blocks(k), n), dtype=torch.float32, device=device).t() if rows == 1 else torch.empty((_blocks(n), _blocks(k)), dtype=torch.float32, device=device)
    _check(_ffi.lib().triteia_hip_fp8_quantize(_ffi.ptr(x), x.stride(0), n, k, rows, _ffi.ptr(codes), k, _ffi.ptr(scales), *scales.stride(),
                                               int(x.dtype == torch.bfloat16), _ffi.device_index(x), _ffi.stream_of(x)))
    return codes, scales


def dequantize_fp8(codes, scales, dtype):
    out = native().dequantize_fp8(codes, scales, dtype)
    if out is not None:
        return out
    device = _require(codes=codes, scales=scales)
    if codes.dtype != torch.float8_e4m3fn or codes.dim() != 2:
        raise RuntimeError(f"codes must be [rows, elements] in torch.float8_e4m3fn, got {tuple(codes.shape)} in {codes.dtype}")
    if dtype not in _TYPES:
        raise RuntimeError(f"values in {dtype}: torch.float16, torch.bfloat16 or torch.float32")
    n, k = codes.shape
    _width("codes", k)
    rows = 1 if scales.dim() and scales.shape[0] == n else BLOCK
    scales, codes = _scales("scales", scales, n if rows == 1 else _blocks(n), k), _adjacent(codes, n)
    out = torch.empty((n, k), dtype=dtype, device=device)
    _check(_ffi.lib().triteia_hip_fp8_values(_ffi.ptr(codes), codes.stride(0), _ffi.ptr(scales), *scales.stride(), rows, n, k, _ffi.ptr(out), _TYPES[dtype],
                                             _ffi.device_index(codes), _ffi.stream_of(codes)))
    return out


def matmul_fp8(x, weight, weight_scale, x_scale, dtype):
    out = native().matmul_fp8(x, weight, weight_scale, x_scale, dtype)
    if out is not None:
        return out
    device = _require(optional=("x_scale",), x=x, weight=weight, weight_scale=weight_scale, x_scale=x_scale)
    if weight.dtype != torch.float8_e4m3fn or weight.dim() != 2:
        raise RuntimeError(f"weight must be [features, elements] in torch.float8_e4m3fn, got {tuple(weight.shape)} in {weight.dtype}")
    m, k = weight.shape
    _width("weight", k)
    w_stride = weight.stride(0) if m > 1 else k                        # (a single row's may be any number)
    if m and (weight.stride(1) != 1 or not 0 <= w_stride <= 1 << 24 or w_stride % 16 or weight.data_ptr() % 16 or weight.is_neg()):
        raise RuntimeError(f"weight's rows must be of adjacent elements, start on 16 bytes and lie up to 2^24 elements apart, got strides {weight.stride()}")
    weight_scale = _scales("weight_scale", weight_scale, _blocks(m), k)
    codes = x.dtype == torch.float8_e4m3fn
    if not codes and x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"x must be in torch.float16, torch.bfloat16 or torch.float8_e4m3fn, got {x.dtype}")
    if codes != (x_scale is not None):
        raise RuntimeError("x_scale belongs to an x in torch.float8_e4m3fn")
    if x.dim() < 1 or x.shape[-1] != k:
        raise RuntimeError(f"x has shape {tuple(x.shape)}, expected rows of {k}")
    dtype = dtype or (torch.float16 if codes else x.dtype)
    if dtype not in _TYPES:
        raise RuntimeError(f"a product in {dtype}: torch.float16, torch.bfloat16 or torch.float32")
    shape = (*x.shape[:-1], m)
    tokens = x.numel() // k
    if codes and x_scale.shape[:-1] == x.shape[:-1] and x_scale.dim() != 2:
        x_scale = x_scale.reshape(tokens, x_scale.shape[-1])
    if codes:
        x_scale = _scales("x_scale", x_scale, tokens, k)
    x = _adjacent(x, tokens)
    out = torch.empty(shape, dtype=dtype, device=device)
    x_type = 2 if codes else _TYPES[x.dtype]
    nbytes = _ffi.lib().triteia_hip_fp8_scratch_bytes(tokens, m, k, x_type)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _check(_ffi.lib().triteia_hip_fp8_matmul(
        _ffi.ptr(x), x.stride(0), x_type, _ffi.ptr(x_scale), *(x_scale.stride() if codes else (0, 0)), _ffi.ptr(weight), w_stride, _ffi.ptr(weight_scale),
        *weight_scale.stride(), _ffi.ptr(out), _TYPES[dtype], tokens, m, k, _ffi.ptr(scratch), nbytes, _ffi.device_index(x), _ffi.stream_of(x)))
    return out
