"""The policy loss's sum of weights at numbers of rows on both sides of where one
wave adds them up by itself, one workgroup and several do.  Bounds as in
test_gpu_policy_loss.py."""

import pytest
import torch

from conftest import announce
from oracle import token_rows as orow
from test_gpu_policy_loss import _compare, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["step", "train"])
@pytest.mark.parametrize("kind", ["none", "bool", "weights"])
@pytest.mark.parametrize("rows", [63, 64, 65, 256, 257, 511, 512, 513, 4096, 4097, 9000])
def test_sum_of_weights(rows, kind, how):
    announce(f"policy_loss sum of weights {rows} {kind} {how}")
    g, x, labels, old, ref, adv = _inputs(1, rows, 21, torch.float32, seed=rows)
    labels[0, torch.rand(rows, generator=g) < 0.1] = orow.IGNORE
    mask = None
    if kind != "none":
        mask = torch.rand(1, rows, generator=g)
        mask = mask < 0.6 if kind == "bool" else mask * (mask < 0.8)
        if kind == "weights":
            mask[labels == orow.IGNORE] = float("nan")  # not looked at
    got = _run(x, labels, old, ref, adv, mask, 0.05, how)
    if kind == "weights":
        mask = torch.where(labels == orow.IGNORE, 0.0, mask)
    _compare(x, labels, old, ref, adv, mask, 0.05, got)


@pytest.mark.parametrize("how", ["step", "train"])
def test_ratio_of_small_probabilities(how):
    """A token's log-probability of -40 has 32-bit neighbours 3.8e-6 apart; its ratio to the old
    one's is as exact as exp.  With the advantage 1 and within the clip it is the loss, but for its
    sign: the sum of exponentials is 2 to 1e-17, and what is rounded is the difference (at most
    0.1), its exp (two units with its argument's product) and three products."""
    announce(f"policy_loss ratio of small probabilities {how}")
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    g = torch.Generator().manual_seed(5)
    for _ in range(24):
        x = torch.tensor([[0.0, -39.0, -60.0, 0.0]]) - torch.tensor([[0.0, 1.0, 0.0, 0.0]]) * \
            torch.rand(1, generator=g)
        old = x[0, 1:2] - 0.693 + 0.1 * torch.rand(1, generator=g)
        args = (torch.tensor([1]).cuda(), old.cuda(), torch.ones(1).cuda())
        if how == "step":
            loss = policy_loss_and_grad(x.cuda(), *args)[0]
        else:
            loss = policy_loss(x.cuda().requires_grad_(True), *args)[0].detach()
        want = -torch.exp(orow.logp(x, torch.tensor([1]))[0] - old.double()[0])
        assert abs(loss.item() / want.item() - 1) <= 8 * 2.0 ** -24
