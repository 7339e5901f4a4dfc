"""Error bounds of the row operators, from the arithmetic the kernels use.

u = 2^-24.  Of a row with exponents t_v = (x_v - m) / tau <= 0 and p = softmax:

* an exponential is off by a relative u (3 |t| + 3): the difference, the product
  with log2(e) / tau (a constant and a product of one rounding each), and the
  instruction, of one unit, where results below 2^-126 may be flushed to 0;
* their sum by the mean of that and by u a term added one after the other: at
  most V, and no more than V / 64 + 64 where lanes share a row;
* log S by the relative error of S, u log S and the instruction's u; logp by
  that, u (2 |t_label| + 2) for the label's term, and a rounding u |logp|.

dlogits follows from exp, S, and the coefficient's own error, rounded once.
"""

import torch

U = 2.0 ** -24
# half a unit in the last of 24, 8 and 11 bits, relative to the smallest number that has them
TYPE_EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPE_TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _terms(x, temperature):
    x = x.double() / temperature
    t = (x - x.max(1, keepdim=True).values).clamp(min=-1e5)
    e = torch.exp(t)
    s = e.sum(1)
    mean = (e * t.abs()).sum(1) / s
    return t, s, mean, min(x.shape[1], x.shape[1] // 64 + 64)


def sum_error(x, temperature=1.0):
    """Relative error of S, a row."""
    _, _, mean, adds = _terms(x, temperature)
    return U * (3 * mean + adds + 8)


def logp_error(x, labels, logp, temperature=1.0):
    t, s, _, _ = _terms(x, temperature)
    lab = labels.clamp(0, x.shape[1] - 1)
    tl = t.gather(1, lab[:, None])[:, 0].abs()
    return sum_error(x, temperature) + U * (2 * tl + 2 * torch.log(s) + 6 + 2 * logp.abs())


def dlogits_error(x, labels, coef, coef_err, want, dtype, temperature=1.0):
    """Elementwise bound for dlogits = coef / tau (onehot - p)."""
    t, _, _, _ = _terms(x, temperature)
    p = torch.exp(t) / torch.exp(t).sum(1, keepdim=True)
    c = coef.double().abs()[:, None] / temperature
    rel = sum_error(x, temperature)[:, None] + U * (3 * t.abs() + 10)
    one = torch.zeros_like(p)
    one.scatter_(1, labels.clamp(0, x.shape[1] - 1)[:, None], 1.0)
    err = c * (p * rel + one * 4 * U) + coef_err.double()[:, None] / temperature * (p + one)
    return err + (want.abs() + err) * TYPE_EPS[dtype] + TYPE_TINY[dtype] * 4 + c * 2.0 ** -125
