"""Matrices in 8-bit floating point (e4m3) with a scale for each block of 128
numbers: the layouts that the norm, the quantisers and the product share.

Codes are a float8_e4m3fn tensor whose rows lie a multiple of 16 bytes apart.
Scales are float32, or powers of two as float8_e8m0fnu; those of rows,
[..., blocks], are a view of memory with the blocks first, so that the scales of
one block lie next to each other, row after row.
"""

import torch

from framework import capi

BLOCK = 128
CODES = torch.float8_e4m3fn
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SCALES = {torch.float32: 0, torch.float8_e8m0fnu: 1}


def require_scales(scale_dtype):
    capi.require(scale_dtype in SCALES, "scale_dtype must be torch.float32 or torch.float8_e8m0fnu")


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def pitch(n):
    """Bytes between rows of n codes."""
    return (n + 15) // 16 * 16


def new_codes(like, lead, n):
    """Codes [*lead, n] on the GPU of ``like``, and the bytes between their rows."""
    p = (n + 15) // 16 * 16
    codes = like.new_empty(*lead, p, dtype=CODES)
    return (codes if p == n else codes[..., :n]), p


def new_scales(like, lead, n, dtype):
    """Scales of rows of n numbers, [*lead, blocks]."""
    n = (n + 127) // 128
    if len(lead) == 1:
        rows = lead[0]
        return like.new_empty_strided((rows, n), (1, rows), dtype=dtype)
    return like.new_empty(n, *lead, dtype=dtype).movedim(0, -1)


def rows_of(x):
    """(x, rows, numbers a row, numbers between rows) with dense rows, copied only if it must be."""
    D = x.shape[-1]
    if not x.is_contiguous():
        if x.dim() == 2 and (D == 1 or x.stride(1) == 1):
            return x, x.shape[0], D, x.stride(0)
        x = x.contiguous()
    return x, x.numel() // D, D, D
