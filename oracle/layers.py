"""CPU oracle of the 8-bit layers' operators -- TEST INFRASTRUCTURE ONLY.

  * ``to_e4m3``: a number's nearest e4m3 one, by arithmetic on its exponent;
  * ``quantize``: codes (as numbers) and scales of blocks, in the operators' own
    32-bit steps, which are single IEEE operations: equal to the last bit;
  * ``matmul`` and ``norm`` / ``norm_backward``: the definitions in float64.

Pinned by tests/test_oracle_layers.py.
"""

import numpy as np
import torch

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126


def to_e4m3(v):
    """float64 array -> the e4m3 numbers nearest, ties to even; NaN past 464."""
    v = np.asarray(v, dtype=np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.abs(v)))
        e = np.where(2.0 ** e > np.abs(v), e - 1, e)      # log2 may round up to a whole number
        e = np.clip(e, -6, 8)
        step = 2.0 ** (e - 3)
        q = np.rint(v / step) * step
    q = np.where(np.abs(v) > 464.0, np.nan, np.where(np.abs(q) > TOP, np.copysign(TOP, v), q))
    return np.where(np.abs(v) == 464.0, np.nan, np.where(v == 0, v, q))


def scale_of(a, power2):
    """Scales (float64) of largest magnitudes a (float32 array)."""
    a = np.asarray(a, dtype=np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.maximum(a / np.float32(TOP), np.float32(LEAST))
    if not power2:
        return s.astype(np.float64)
    out = np.empty(a.shape, dtype=np.float64)
    for i, x in np.ndenumerate(a):
        if np.isinf(x):
            out[i] = np.nan
            continue
        k = -126
        while TOP * 2.0 ** k < float(x):
            k += 1
        out[i] = 2.0 ** k
    return out


def quantize(x, tiles=False, power2=False):
    """(codes as float64 [M, K], scales float64) of x [M, K], any torch float type."""
    x = x.detach().cpu().float().numpy()
    M, K = x.shape
    p = BLOCK if tiles else 1
    mb, kb = -(-M // p), -(-K // BLOCK)
    codes = np.empty((M, K))
    a = np.zeros((mb, kb), dtype=np.float32)
    for i in range(mb):
        for j in range(kb):
            block = np.abs(x[i * p:(i + 1) * p, j * BLOCK:(j + 1) * BLOCK])
            block = block[~np.isnan(block)]
            a[i, j] = block.max() if block.size else 0.0
    s = scale_of(a, power2)
    with np.errstate(all="ignore"):
        inverse = (np.float32(1.0) / s.astype(np.float32))
        inverse = np.where(np.isnan(s), np.float32(0), inverse)
        each = inverse.repeat(p, 0)[:M].repeat(BLOCK, 1)[:, :K]
        codes = to_e4m3((x * each).astype(np.float64))
    return torch.from_numpy(codes), torch.from_numpy(s)


def spread(scales, M, K):
    """A scale for each of [M, K] numbers, of rows' or tiles' scales."""
    s = scales.double()
    if s.shape[0] != M:
        s = s.repeat_interleave(BLOCK, 0)[:M]
    return s.repeat_interleave(BLOCK, 1)[:, :K]


def values(codes, scales):
    """What codes and scales stand for, float64."""
    codes = codes.double() if codes.dtype == torch.float64 else codes.float().double()
    return codes * spread(scales if scales.dtype == torch.float64 else scales.float(), *codes.shape)


def matmul(a, b):
    """(a b^T, |a| |b|^T) of float64 matrices."""
    return a @ b.t(), a.abs() @ b.abs().t()


def norm(x, weight, residual=None, eps=1e-6):
    """(y, h, 1 / rms) in float64; h rounded to the residual's type."""
    h = x.double()
    if residual is not None:
        h = (x.float() + residual.float()).to(residual.dtype).double()
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * r * weight.double(), h, r


def norm_backward(dy, h, weight, r, dh=None):
    """(dx, dweight) in float64 of rows [M, D]."""
    d, u = dy.double(), h * r
    g = d * weight.double()
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return dx, (d * u).sum(0)
