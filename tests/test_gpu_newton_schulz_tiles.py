"""Sizes whose products take each of the tile shapes, whole tiles and not, one
matrix and many, and X X' summed in parts.  Against the iteration in 64 bits on
the GPU; the bound is four times what roundings of the kernels' operands move
it by, and the rounding to the result's type."""

import pytest
import torch

from conftest import announce
from oracle import newton_schulz as ons

pytestmark = pytest.mark.gpu

OPERAND = {"half": 2.0 ** -11, "full": 2.0 ** -21}


# tiles of 256 and 192; 192 and 128; 128; 64; 64 in parts
@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("count,m,n", [(1, 4096, 4096), (1, 4000, 4133), (16, 768, 768),
                                       (3, 2100, 1500), (4, 1000, 2731), (1, 700, 650),
                                       (1, 300, 8192), (2, 6001, 129), (1, 1024, 1408)])
def test_tiles(count, m, n, precision):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz {count} x {m} x {n} {precision}")
    g = torch.Generator(device="cuda").manual_seed(m + n)
    r = min(m, n) // 4
    G = (torch.randn(count, m, r, generator=g, device="cuda") @
         torch.randn(count, r, n, generator=g, device="cuda") / r ** 0.5 +
         0.3 * torch.randn(count, m, n, generator=g, device="cuda"))
    out = newton_schulz(G, precision=precision)
    again = newton_schulz(G, precision=precision)
    assert torch.equal(out, again)
    for i in {0, count - 1}:
        want = ons.by_products(G[i])
        off = ons.by_products(G[i], operand=OPERAND[precision], product=2.0 ** -22, seed=1)
        bound = 4 * (off - want).norm() + 2.0 ** -24 * want.norm()
        assert (out[i].double() - want).norm() <= bound
        # and no element far out, as a tile written to the wrong place would be
        assert (out[i].double() - want).abs().max() <= 64 * (off - want).abs().max()
