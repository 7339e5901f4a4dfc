"""Central differences of the norm, and how far they may be from its gradients.

For f = sum(dy y) + sum(dh h), a coordinate's difference quotient d over `step`
and its gradient g, computed in 32 bits, against the same in 64 (D, G):

    |d - g| <= |d - D| + |D - G| + |G - g|

|D - G| is the step's truncation, known in 64 bits.  h is exact (the numbers are
whole multiples of the step, few bits wide), so d is off by what two values of y
are, sum(|dy| error of y) / step at most.  The last term is the gradient's own bound.
"""

import torch

import layer_tolerances as tol
from oracle import layers as ol

STEP = 2.0 ** -6
EPS = 1e-5


def inputs(rows, d, seed):
    """x, residual, weight, dy, dh in float32: multiples of the step up to 2."""
    g = torch.Generator().manual_seed(seed)

    def whole(*shape):
        return torch.randint(-128, 129, shape, generator=g).float() * STEP
    return whole(rows, d), whole(rows, d), 1 + whole(d) / 4, whole(rows, d), whole(rows, d)


def moves(rows, d):
    """(which input, index): every coordinate of x and of the weight."""
    return [("x", (i, j)) for i in range(rows) for j in range(d)] + \
        [("weight", (j,)) for j in range(d)]


def moved(x, w, which, at, by):
    x, w = x.clone(), w.clone()
    (x if which == "x" else w)[at] += by
    return x, w


def bounds(x, res, w, dy, dh):
    """{(which, index): (D, bound of |d - g|)}."""
    _, wh, r = ol.norm(x, w, res, EPS)
    dx, dw = ol.norm_backward(dy, wh, w, r, dh)
    err_dx = tol.dx_error(dy, wh, w, r, dh, dx, torch.float32)
    err_dw = tol.dw_error(dy, wh, r, dw, torch.float32)
    out = {}
    for which, at in moves(*x.shape):
        f, err = [], 0.0
        for by in (STEP, -STEP):
            y, h, _ = ol.norm(*(moved(x, w, which, at, by)), res, EPS)
            f.append((y * dy).sum() + (h * dh).sum())
            err += (tol.y_error(y, torch.float32) * dy.abs()).sum()
        d = (f[0] - f[1]) / (2 * STEP)
        g, own = (dx[at], err_dx[at]) if which == "x" else (dw[at], err_dw[at])
        out[which, at] = d, (err / (2 * STEP) + (d - g).abs() + own).item()
    return out
