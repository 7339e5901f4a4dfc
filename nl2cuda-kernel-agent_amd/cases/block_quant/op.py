"""Matrices in 8-bit floating point with a scale for each block of 128 numbers:
wrapper over the HIP library (kernels/block_quant.hip).

``quantize_rows`` takes activations and gradients, whose blocks are 128 numbers
of a row; ``quantize_tiles`` weights, whose blocks are 128 rows by 128 columns.
Either gives the transposed matrix too, from the same reading, for the products
of a backward.  There is no CPU path: without a GPU the library refuses to load.
"""

import functools
import os

import torch

from framework import capi, e4m3
from framework.loader import load_kernel

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "block_quant_hip"
SOURCES = ["block_quant.hip"]


def bind_library(lib):
    V, I64, I = capi.c_void_p, capi.c_int64, capi.c_int
    capi.bind(lib, "block_quant_rows", [V, I, I64, V, I64, V, V, I64, V, I, I64, I64, V])
    capi.bind(lib, "block_quant_tiles", [V, I, I64, V, I64, V, V, I64, I, I64, I64, V])
    capi.bind_last_error(lib, "block_quant_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


def _check(x, scale_dtype):
    capi.require(x.is_cuda, "x must be a GPU tensor")
    capi.require(x.dtype in e4m3.DTYPES, "x must be float32, bfloat16 or float16")
    e4m3.require_scales(scale_dtype)


def quantize_rows(x, scale_dtype=torch.float8_e8m0fnu, transposed=False):
    """(codes, scales) of x [..., K]: float8_e4m3fn [..., K], and a scale for each
    128 numbers of a row, [..., ceil(K / 128)]; without a gradient.

    A block's scale is its largest magnitude / 448 as float32, or the least
    power of two that is no smaller as float8_e8m0fnu, never below 2^-126.

    transposed: x is [M, K], and (codes, scales, codes_t, scales_t) come back,
    codes_t [K, M] with blocks along M, scales_t [K, ceil(M / 128)].
    """
    _check(x, scale_dtype)
    capi.require(x.dim() >= 1 and x.size(-1) >= 1, "x must be [..., K] with K >= 1")
    capi.require(not transposed or x.dim() == 2, "x must be [M, K] to be transposed")
    lib = _lib()
    x = x.detach()
    lead = x.shape[:-1]
    x, M, K, stride = e4m3.rows_of(x)
    codes, pitch = e4m3.new_codes(x, lead, K)
    scales = e4m3.new_scales(x, lead, K, scale_dtype)
    codes_t = scales_t = None
    pitch_t = 0
    if transposed:
        codes_t, pitch_t = e4m3.new_codes(x, (K,), M)
        scales_t = e4m3.new_scales(x, (K,), M, scale_dtype)
    st = capi.launch(lib.block_quant_rows, x.get_device(), x.data_ptr(), e4m3.DTYPES[x.dtype],
                     stride, codes.data_ptr(), pitch, scales.data_ptr(),
                     codes_t.data_ptr() if transposed else 0, pitch_t,
                     scales_t.data_ptr() if transposed else 0, e4m3.SCALES[scale_dtype], M, K)
    if st:
        capi.check(st, lib.block_quant_last_error, "quantize_rows")
    return (codes, scales, codes_t, scales_t) if transposed else (codes, scales)


def quantize_tiles(w, scale_dtype=torch.float8_e8m0fnu, transposed=False):
    """(codes, scales) of w [N, K]: float8_e4m3fn [N, K], and a scale for each tile of
    128 x 128, [ceil(N / 128), ceil(K / 128)], as in ``quantize_rows``; without a
    gradient.

    transposed: (codes, scales, codes_t, scales_t) come back, the same codes as
    [K, N] and the transposed view of the scales.
    """
    _check(w, scale_dtype)
    capi.require(w.dim() == 2 and w.size(1) >= 1, "w must be [N, K] with K >= 1")
    lib = _lib()
    w, N, K, stride = e4m3.rows_of(w.detach())
    codes, pitch = e4m3.new_codes(w, (N,), K)
    scales = w.new_empty((e4m3.blocks(N), e4m3.blocks(K)), dtype=scale_dtype)
    codes_t, pitch_t = e4m3.new_codes(w, (K,), N) if transposed else (None, 0)
    st = capi.launch(lib.block_quant_tiles, w.get_device(), w.data_ptr(), e4m3.DTYPES[w.dtype],
                     stride, codes.data_ptr(), pitch, scales.data_ptr(),
                     codes_t.data_ptr() if transposed else 0, pitch_t, e4m3.SCALES[scale_dtype],
                     N, K)
    if st:
        capi.check(st, lib.block_quant_last_error, "quantize_tiles")
    return (codes, scales, codes_t, scales.t()) if transposed else (codes, scales)


def candidate(inputs, params):
    """Framework candidate contract: inputs={"X"} -> what its codes and scales stand for."""
    codes, scales = quantize_rows(inputs["X"], params.get("scale_dtype", torch.float8_e8m0fnu))
    each = scales.float().repeat_interleave(e4m3.BLOCK, -1)[..., :codes.size(-1)]
    return codes.float() * each


forward_only = candidate
