"""The training operators as programs use them beyond a plain call: the
precision that nobody asked for, autograd's hooks and version counters, saved
optimisers, operands that share memory.  Tests that need no GPU put a recorder
in the place of the library call."""

import pytest
import torch

from conftest import announce
from oracle import newton_schulz as ons


def _matrix(m, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 4)
    return (torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) / r ** 0.5
            + 0.3 * torch.randn(m, n, generator=g))


# ------------------------------------------- Newton-Schulz: bits of the iterates
def _within_a_rounding(got, want, iterates, eps, factor=1.0):
    """got = want rounded to its type, `iterates` further off at most.  What roundings of the full
    iterates' size move the result by is in the norm: no element is off by more than all."""
    slack = factor * 4 * iterates.norm()
    assert torch.all((got.cpu().double() - want).abs() <= eps * 1.01 * want.abs() + slack + 2.0 ** -25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,eps", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("m,n", [(150, 200), (300, 130)])
def test_16_bit_matrices_are_iterated_in_full(m, n, dtype, eps):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz of 16 bits, no precision given {m} x {n} {dtype}")
    G = _matrix(m, n).to(dtype)
    got = newton_schulz(G.cuda())
    assert torch.equal(got, newton_schulz(G.cuda(), precision="full"))
    want = ons.orthogonalise(G)
    off = ons.by_products(G, operand=2.0 ** -21, product=2.0 ** -22, seed=1)
    _within_a_rounding(got, want, off - want, eps)


@pytest.mark.gpu
def test_16_bit_weights_are_updated_from_full_iterates():
    from cases.newton_schulz.op import muon_step
    announce("muon_step of 16-bit weights, no precision given")
    W, G = (0.02 * _matrix(150, 200, 1)).bfloat16(), _matrix(150, 200, 2)
    Wd, Md = W.cuda(), torch.zeros(150, 200, device="cuda")
    full, Mf = W.cuda(), Md.clone()
    muon_step(Wd, G.cuda(), Md, lr=0.05, nesterov=False)
    muon_step(full, G.cuda(), Mf, lr=0.05, nesterov=False, precision="full")
    assert torch.equal(Wd, full)
    O = ons.orthogonalise(G)
    off = ons.by_products(G, operand=2.0 ** -21, product=2.0 ** -22, seed=1) - O
    _within_a_rounding(Wd, W.double() - 0.05 * O, off, 2.0 ** -8, 0.05)
