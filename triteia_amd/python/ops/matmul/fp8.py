"""The base weight that all variants share, in 8 bits: e4m3 with a scale for each block of 128 x 128, multiplied on the matrix cores with activations that have a
scale for every token and 128 channels.  (The reference's form, ops/matmul/fp8.py:9-43, has one scale for a whole tensor.)"""
import torch

from triteia_amd.python import capi

__all__ = ["quantize_fp8", "dequantize_fp8", "matmul_fp8"]


def quantize_fp8(x, rows=1):
    """(codes, scales) of x [n, k] in fp16 or bf16: e4m3 codes [n, k] and float32 scales [n, k / 128] (rounded up; rows=1: activations) or [n / 128, k / 128] (rows=128:
    weights).  value = code * scale, scale = max|x| of the block / 448, code = x / scale to the nearest.  A block of magnitudes below 1e-30 is zeros; one that holds an
    infinity or a NaN reads back as NaN.  k is a multiple of 16.  Serving only: no gradient is recorded.

    Scales of rows=1 come as a transposed view, a block's of all rows adjacent, as `matmul_fp8` reads them best; it takes any other strides too."""
    return capi.quantize_fp8(x, rows)


def dequantize_fp8(codes, scales, dtype=torch.float16):
    """The values of `quantize_fp8`'s codes [n, k], in fp16, bf16 or fp32; scales for single rows or for 128 of them."""
    return capi.dequantize_fp8(codes, scales, dtype)


def matmul_fp8(x, weight, weight_scale, x_scale=None, dtype=None):
    """x [..., k] @ weight^T -> [..., m]: weight [m, k] in e4m3 with weight_scale [m / 128, k / 128] (rounded up), as `quantize_fp8(w, rows=128)` leaves them.

    x in fp16 or bf16 is quantised in the call, with a scale for every token and 128 elements; in e4m3 it comes with such an x_scale [..., k / 128].
    Products of eight adjacent codes are added by the matrix cores in fixed point, each without what lies below 2^-13 of the largest of the eight (together up to 7 2^-13 of that product, also
    where the large ones cancel: 448 * 448 - 448 * 448 + 2 * 2 is 0); all else is added in 32 bits and rounded once, to `dtype`: fp16, bf16 or fp32 (None: x's, or fp16 for an x in e4m3).
    Random codes come out 1.3e-5 off in norm, beside the 2e-2 by which the codes are off what they stand for.  k is a multiple of 16, m and the tokens are any number;
    weight's rows start on 16 bytes.  Serving only: no gradient is recorded."""
    return capi.matmul_fp8(x, weight, weight_scale, x_scale, dtype)
