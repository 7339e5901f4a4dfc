"""Row operators on logits of tens and hundreds of MiB, which go through the
caches in other ways and in another order than small ones: every row's answers
are those, bit for bit, that it gets in a call of 48 MiB of rows, whose answers
other tests compare with the oracle.  Each width takes one number of lanes a row
at any number of rows."""

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

# MiB of logits: both sides of each size at which the use of the caches changes
SIZES = [60, 70, 150, 170, 370, 400]
WIDTHS = [(1001, torch.bfloat16), (2500, torch.float32), (7001, torch.float16)]
PIECE = 48 << 20


def _inputs(mib, v, dtype):
    rows = (mib << 20) // (v * dtype.itemsize)
    g = torch.Generator(device="cuda").manual_seed(v + mib)
    x = torch.randn(rows, v, generator=g, device="cuda", dtype=dtype) * 3
    labels = torch.randint(0, v, (rows,), generator=g, device="cuda")
    labels[torch.rand(rows, generator=g, device="cuda") < 0.2] = -100
    labels[::777] = v - 1
    up = torch.randn(rows, generator=g, device="cuda")
    step = PIECE // (v * dtype.itemsize)
    return x, labels, up, [slice(i, i + step) for i in range(0, rows, step)]


@pytest.mark.parametrize("v,dtype", WIDTHS, ids=str)
@pytest.mark.parametrize("mib", SIZES)
def test_token_logp(mib, v, dtype):
    from cases.token_logp.op import token_logp
    announce(f"token_logp {mib} MiB of {v} {dtype}")
    x, labels, up, pieces = _inputs(mib, v, dtype)

    def both(rows):
        xr = x[rows].detach().requires_grad_(True)
        logp = token_logp(xr, labels[rows])
        (d,) = torch.autograd.grad(logp, xr, up[rows])
        return logp.detach(), d

    logp, d = both(slice(None))
    assert torch.equal(token_logp(x, labels), logp)
    for rows in pieces:
        lp, dp = both(rows)
        assert torch.equal(lp, logp[rows]) and torch.equal(dp, d[rows])


@pytest.mark.parametrize("v,dtype", WIDTHS + [(50257, torch.float32), (140001, torch.bfloat16)],
                         ids=str)
@pytest.mark.parametrize("mib", SIZES)
def test_policy_loss(mib, v, dtype):
    from cases.policy_loss.op import policy_loss_and_grad
    announce(f"policy_loss {mib} MiB of {v} {dtype}")
    x, labels, adv, pieces = _inputs(mib, v, dtype)
    old = torch.full_like(adv, -float(torch.tensor(v).log()) - 4)

    def both(rows, inplace=False):
        xr = x[rows].clone() if inplace else x[rows]
        return policy_loss_and_grad(xr, labels[rows], old[rows], adv[rows], denom=1000.0,
                                    inplace=inplace)[1:]

    logp, d = both(slice(None))
    for a, b in zip(both(slice(None), inplace=True), (logp, d)):
        assert torch.equal(a, b)
    for rows in pieces:
        lp, dp = both(rows)
        assert torch.equal(lp, logp[rows]) and torch.equal(dp, d[rows])
