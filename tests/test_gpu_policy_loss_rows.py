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
