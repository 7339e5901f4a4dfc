"""The preference loss's mean over many pairs of sequences: as many workgroups,
the last of which takes it.  Against float64 of the sequences' sums that the
call itself returns: each pair's loss is rounded to 24 bits, their mean once
more, and the sums were, which moves a pair's by at most beta times that."""

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("pairs", [1, 2, 255, 256, 257, 3000])
def test_mean(pairs):
    from cases.preference_loss.op import preference_loss, preference_loss_and_grad
    announce(f"preference_loss {pairs} pairs")
    g = torch.Generator(device="cuda").manual_seed(pairs)
    x = 2 * torch.randn(2 * pairs, 5, 33, generator=g, device="cuda")
    labels = torch.randint(0, 33, (2 * pairs, 5), generator=g, device="cuda")
    first = None
    for _ in range(20):
        loss, seq, d = preference_loss_and_grad(x, labels, beta=0.3, label_smoothing=0.1)
        first = first or (loss.item(), d)
        assert loss.item() == first[0] and torch.equal(d, first[1])
    assert preference_loss(x, labels, beta=0.3, label_smoothing=0.1)[0].item() == first[0]
    h = 0.3 * seq.double()
    diff = h[:pairs] - h[pairs:]
    sp = torch.nn.functional.softplus
    want = (0.9 * sp(-diff) + 0.1 * sp(diff)).mean()
    bound = 2 * U * want + 0.3 * 2 * U * seq.double().abs().max()
    assert abs(loss.double() - want) <= bound


def test_no_tokens():
    from cases.preference_loss.op import preference_loss_and_grad
    announce("preference_loss without tokens")
    x = torch.empty(6, 0, 9, device="cuda")
    for _ in range(3):
        loss, seq, d = preference_loss_and_grad(x, torch.empty(6, 0, dtype=torch.int64,
                                                               device="cuda"))
        assert abs(loss.item() - 0.6931471805599453) <= 2 * U and not seq.any()
        assert d.shape == x.shape
