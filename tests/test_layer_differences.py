"""The comparison of the norm's gradients with differences rejects wrong gradients:
mistakes planted in the 64-bit formulas, on the CPU."""

import pytest

import layer_differences as ld
from oracle import layers as ol

MISTAKES = {
    "no projection": lambda g, u, r, dh: r * g + dh,
    "no mean": lambda g, u, r, dh: r * (g - u * (g * u).sum(-1, keepdim=True)) + dh,
    "halved": lambda g, u, r, dh: (r * (g - u * (g * u).mean(-1, keepdim=True)) + dh) / 2,
    "zero": lambda g, u, r, dh: 0 * g,
    "no dh": lambda g, u, r, dh: r * (g - u * (g * u).mean(-1, keepdim=True)),
    "r twice": lambda g, u, r, dh: r * r * (g - u * (g * u).mean(-1, keepdim=True)) + dh,
}


@pytest.mark.parametrize("d", [4, 7])
def test_right_gradients_pass_and_wrong_ones_do_not(d):
    x, res, w, dy, dh = ld.inputs(2, d, d)
    _, h, r = ol.norm(x, w, res, ld.EPS)
    u, dy, dh = h * r, dy.double(), dh.double()
    g = dy * w.double()
    bounds = ld.bounds(x, res, w, dy, dh)
    dx, dw = ol.norm_backward(dy, h, w, r, dh)

    def wrong(which, grad):
        return [k for k, (diff, bound) in bounds.items()
                if k[0] == which and abs(diff - grad[k[1]]) > bound]
    assert not wrong("x", dx) and not wrong("weight", dw)
    for name, mistake in MISTAKES.items():
        assert len(wrong("x", mistake(g, u, r, dh))) >= d, name       # half of them or more
    for name, grad in (("halved", dw / 2), ("no r", (dy * h).sum(0)), ("one row", (dy * u)[0]),
                       ("with the weight", dw * w.double()), ("zero", 0 * dw)):
        assert len(wrong("weight", grad)) >= d // 2, name
