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


def new_codes(lead, n, device):
    """Codes [*lead, n] and the bytes between their rows."""
    p = pitch(n)
    codes = torch.empty((*lead, p), dtype=CODES, device=device)
    return (codes if p == n else codes[..., :n]), p


def new_scales(lead, n, dtype, device):
    """Scales of rows of n numbers, [*lead, blocks]."""
    scales = torch.empty((blocks(n), *lead), dtype=dtype, device=device)
    return scales.t() if len(lead) == 1 else scales.movedim(0, -1)


def rows_of(x):
    """(x, rows, numbers a row, numbers between rows) with dense rows, copied only if it must be."""
    D, d = x.size(-1), x.dim()
    dense = D == 1 or x.stride(-1) == 1
    if d == 2 and dense and x.stride(0) >= 0:
        return x, x.size(0), D, x.stride(0)
    if d == 1 and dense:
        return x, 1, D, D
    x = x.contiguous()
    return x, x.numel() // D if D else 0, D, D
