"""Pins the float64 oracles of the training operators: autograd of the losses'
expressions, central differences, closed forms, and planted mistakes that the
comparisons must catch."""

import math

import pytest
import torch

from oracle import newton_schulz as ons
from oracle import token_rows as orow


def _rows(seed, rows=7, v=11):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g, dtype=torch.float64) * 2
    labels = torch.randint(0, v, (rows,), generator=g)
    labels[2] = orow.IGNORE
    return g, x, labels


def test_logp_closed_forms():
    x = torch.zeros(2, 5, dtype=torch.float64)
    assert torch.allclose(orow.logp(x, torch.tensor([0, 4])),
                          torch.full((2,), -math.log(5), dtype=torch.float64))
    x[0, 1] = 3.0
    assert math.isclose(orow.logp(x, torch.tensor([1, orow.IGNORE]), 2.0)[0].item(),
                        1.5 - math.log(4 + math.exp(1.5)))
    assert orow.logp(x, torch.tensor([1, orow.IGNORE]))[1] == 0


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_logp_and_gradient_against_autograd(temperature):
    g, x, labels = _rows(1)
    up = torch.randn(7, generator=g, dtype=torch.float64)
    x.requires_grad_(True)
    keep = labels != orow.IGNORE
    want = torch.log_softmax(x / temperature, 1).gather(1, labels.clamp(min=0)[:, None])[:, 0]
    want = torch.where(keep, want, 0.0)
    assert torch.allclose(orow.logp(x.detach(), labels, temperature), want.detach(), atol=1e-14)
    (d,) = torch.autograd.grad(want, x, up)
    assert torch.allclose(orow.dlogits(x.detach(), labels, up, temperature), d, atol=1e-14)


@pytest.mark.parametrize("weights", [False, True])
def test_policy_against_autograd_and_differences(weights):
    g, x, labels = _rows(2, rows=40)
    lp = orow.logp(x, labels)
    old = lp - 0.4 * torch.randn(40, generator=g, dtype=torch.float64)
    ref = lp + 0.3 * torch.randn(40, generator=g, dtype=torch.float64)
    adv = torch.randn(40, generator=g, dtype=torch.float64)
    mask = torch.rand(40, generator=g) < 0.7
    if weights:
        mask = mask * torch.rand(40, generator=g)
    opts = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05)
    loss, coef = orow.policy(lp, labels, old, adv, ref, mask, **opts)

    def value(q):
        w = torch.where(labels != orow.IGNORE, mask.double(), 0.0)
        r = torch.exp(q - old)
        t = -torch.min(r * adv, r.clamp(0.8, 1.3) * adv)
        t = t + 0.05 * (torch.exp(ref - q) - (ref - q) - 1)
        return (w * t).sum() / w.sum()

    q = lp.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(value(q), q)
    assert abs(value(lp) - loss) < 1e-13 and torch.allclose(coef, d, atol=1e-14)
    h = 1e-6
    for i in range(0, 40, 7):
        e = torch.zeros(40, dtype=torch.float64)
        e[i] = h
        diff = (value(lp + e) - value(lp - e)) / (2 * h)
        assert abs(diff - coef[i]) < 1e-8
    # planted mistakes: the clamp ignored, the sign of the KL term
    wrong = orow.policy(lp, labels, old, adv, ref, mask, clip_low=1.0, clip_high=1e9,
                        kl_coef=0.05)[1]
    assert not torch.allclose(wrong, d, atol=1e-6)
    wrong = orow.policy(lp, labels, old, adv, 2 * lp - ref, mask, **opts)[1]
    assert not torch.allclose(wrong, d, atol=1e-6)


def test_policy_of_nothing_is_zero():
    _, x, labels = _rows(3)
    labels[:] = orow.IGNORE
    z = torch.zeros(7, dtype=torch.float64)
    loss, coef = orow.policy(z, labels, z, z)
    assert loss == 0 and coef.abs().sum() == 0


@pytest.mark.parametrize("average", [False, True])
def test_preference_against_autograd(average):
    g, x, labels = _rows(4, rows=40)
    seqs = [torch.arange(0, 9), torch.arange(9, 10), torch.arange(12, 30), torch.arange(30, 40)]
    ref = torch.randn(4, generator=g, dtype=torch.float64)
    lp = orow.logp(x, labels)
    loss, seq, coef = orow.preference(lp, labels, seqs, ref, 0.3, 0.1, average)
    q = lp.clone().requires_grad_(True)
    s = torch.stack([q[i].sum() / (max(1, int((labels[i] != orow.IGNORE).sum())) if average else 1)
                     for i in seqs])
    d = 0.3 * ((s - ref)[:2] - (s - ref)[2:])
    value = (-0.9 * torch.log(torch.sigmoid(d)) - 0.1 * torch.log(torch.sigmoid(-d))).mean()
    (want,) = torch.autograd.grad(value, q)
    assert abs(value - loss) < 1e-13 and torch.allclose(coef, want, atol=1e-14)
    assert torch.allclose(seq, s.detach()) and coef[10:12].abs().sum() == 0


@pytest.mark.parametrize("m,n", [(1, 1), (5, 9), (9, 5), (16, 16)])
def test_newton_schulz_products_follow_the_singular_values(m, n):
    G = torch.randn(m, n, generator=torch.Generator().manual_seed(m * 31 + n))
    a, b = ons.orthogonalise(G), ons.by_products(G)
    assert torch.allclose(a, b, atol=1e-12)
    # a coefficient of another sign, or a step more, must be seen
    assert not torch.allclose(a, ons.by_products(G, (3.4445, 4.7750, 2.0315)), atol=1e-3)
    assert not torch.allclose(a, ons.by_products(G, steps=6), atol=1e-3)


def test_roundings_of_operands_move_the_result_in_proportion():
    G = torch.randn(24, 40, generator=torch.Generator().manual_seed(5))
    exact = ons.by_products(G)
    d = [(ons.by_products(G, operand=s, seed=1) - exact).norm().item() for s in (1e-8, 1e-6)]
    assert 50 < d[1] / d[0] < 200
