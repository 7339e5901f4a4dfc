"""Error bounds of the 8-bit layers' operators, from the arithmetic the kernels use.

u = 2^-24.  Norm of D numbers: a lane adds 8 ceil(D / 8192) to 16 squares one after
the other, then 6 lanes' steps and at most 16 waves: `adds` covers each kernel's.
A mean's relative error is (adds + 2) u, 1 / sqrt adds two units and halves what is
under the root.  Sums over rows: at most rows / 256 + 1 a workgroup, four waves,
1024 / 16 and 16 sums after that.

The product: a block's 128 products and the sum of blocks in 32 bits, each
addition off by at most a unit in the last place (2 u) of a number that the sum of
magnitudes bounds; scales applied afterwards cost three more roundings a block.
For 16-bit results eight products at a time are added in a window that drops what
lies 13 bits below the largest: seven of them are off by 2^-13 of it at most.
"""

import torch

U = 2.0 ** -24
# half a unit in the last of 24, 8 and 11 bits, relative to the smallest number that has them
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def adds(D):
    return 16 + 8 * -(-D // 8192) + 6 + 16


def rounded(err, want, dtype):
    """`err` and a rounding of what it is off from."""
    return err + (want.abs() + err) * EPS[dtype] + TINY[dtype]


def y_error(y, dtype):
    D = y.shape[-1]
    return rounded(y.abs() * U * ((adds(D) + 2) / 2 + 6), y, dtype)


def dx_error(dy, h, weight, r, dh, dx, dtype):
    D = h.shape[-1]
    g, v = (dy.double() * weight.double()).abs(), (h * r).abs()
    size = r * (g + v * (g * v).mean(-1, keepdim=True))
    err = size * U * (2 * (adds(D) + 10) + 10)
    if dh is not None:
        err = err + U * (size + dh.double().abs())
    return rounded(err, dx, dtype)


def dw_error(dy, h, r, dw, dtype):
    rows, D = h.shape
    size = (dy.double() * h * r).abs().sum(0)
    return rounded(size * U * (rows / 256 + 92 + (adds(D) + 2) / 2 + 8), dw, dtype)


def largest_of_eight(a, b):
    """sum over each eight products of a row of a and one of b of the largest.  In float32, of
    rows' numbers over a power of two that brings the operand's largest to 1 to 2: exact, and
    (x / p)(y / q) p q = x y, so that operands beyond float32's range have a bound too."""
    pad = (0, -a.shape[1] % 8)
    tops = [2.0 ** torch.floor(torch.log2(t.abs().max().clamp_min(1e-300))) for t in (a, b)]
    a, b = (torch.nn.functional.pad((t.abs() / top).float(), pad) for t, top in zip((a, b), tops))
    out = torch.empty(a.shape[0], b.shape[0], dtype=torch.float64)
    step = max(1, (1 << 24) // (b.numel() + 1))
    for i in range(0, a.shape[0], step):
        p = a[i:i + step, None] * b
        out[i:i + step] = p.view(*p.shape[:2], -1, 8).amax(-1).double().sum(-1)
    return out * (1 + 2.0 ** -22) * (tops[0] * tops[1])


def matmul_error(a, b, size, want, dtype):
    """For a b^T; size: |a| |b|^T."""
    blocks = -(-a.shape[1] // 128)
    err = size * 2 * U * (128 + 5 * blocks + 16)
    if dtype != torch.float32:
        err = err + 7 * 2.0 ** -13 * largest_of_eight(a, b)
    return rounded(err, want, dtype)
