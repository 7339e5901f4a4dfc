"""The operators together, as the example uses them: a model learns from
rewards, and from pairs of answers."""

import os
import sys

import pytest
import torch

from conftest import PACKAGE, announce

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(PACKAGE, "examples"))


def test_rewards_rise():
    announce("post-training from rewards")
    import post_training as ex
    g = torch.Generator(device="cuda").manual_seed(0)
    model = ex.Model(torch.Generator().manual_seed(0))
    rewards = ex.learn_from_rewards(model, 60, g)
    assert all(torch.isfinite(p).all() for p in model.parameters())
    # one in 48 by chance; the last ten steps far above it
    assert sum(rewards[:3]) / 3 < 0.1 and sum(rewards[-10:]) / 10 > 0.3


def test_pairs_are_told_apart():
    announce("post-training from pairs")
    import post_training as ex
    g = torch.Generator(device="cuda").manual_seed(0)
    model = ex.Model(torch.Generator().manual_seed(1))
    losses = ex.learn_from_pairs(model, 40, g)
    # log 2 before the model has moved
    assert abs(losses[0] - 0.6931) < 1e-3 and losses[-1] < 0.3
