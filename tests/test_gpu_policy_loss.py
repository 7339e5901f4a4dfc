"""The clipped policy loss on the GPU, both ways to its gradient, against the
float64 oracle.  Bounds: operator_tolerances.py for logp and dlogits; a term's
coefficient is off by its derivative times logp's error and u times what it is
made of, the loss by the mean of its terms' errors."""

import math

import pytest
import torch

import operator_tolerances as tol
from conftest import announce
from oracle import token_rows as orow

pytestmark = pytest.mark.gpu

LOW, HIGH = 0.2, 0.28


def _inputs(b, s, v, dtype, seed=0, temperature=1.0):
    g = torch.Generator().manual_seed(seed + 7 * v + s)
    x = (torch.randn(b, s, v, generator=g) * 2).to(dtype)
    labels = torch.randint(0, v, (b, s), generator=g)
    lp = orow.logp(x.reshape(-1, v), labels.reshape(-1), temperature).view(b, s)
    ratio = 0.25 * torch.randn(b, s, generator=g, dtype=torch.float64)
    for edge in (math.log(1 - LOW), math.log(1 + HIGH)):  # not within rounding of an edge
        near = (ratio - edge).abs() < 1e-2
        ratio = torch.where(near, edge + torch.where(ratio < edge, -1e-2, 1e-2), ratio)
    old = (lp - ratio).float()
    ref = (lp + 0.3 * torch.randn(b, s, generator=g)).float()
    adv = torch.randn(b, s, generator=g)
    return g, x, labels, old, ref, adv


def _expect(x, labels, old, ref, adv, mask, kl, temperature, denom=None):
    """(loss, loss bound, logp, coef, coef bound, keep) over flat rows."""
    v = x.shape[-1]
    x, labels, old, adv = x.reshape(-1, v), labels.reshape(-1), old.reshape(-1), adv.reshape(-1)
    ref = None if ref is None else ref.reshape(-1)
    mask = None if mask is None else mask.reshape(-1)
    keep = orow.counted(labels, mask)
    lp = orow.logp(x, labels, temperature, keep)
    loss, coef = orow.policy(lp, labels, old, adv, ref, mask, LOW, HIGH, kl, denom)
    err = tol.logp_error(x, labels, lp, temperature)
    w = keep.double() if mask is None or mask.dtype != torch.float32 else mask.double() * keep
    D = float(denom) if denom else max(float(w.sum()), 1e-300)
    r = torch.exp(lp - old.double())
    e = torch.exp(ref.double() - lp) if kl else torch.zeros_like(lp)
    d = (ref.double() - lp).abs() if kl else torch.zeros_like(lp)
    diff = (lp - old.double()).abs()
    slope = r * adv.double().abs() + kl * (e + 1)
    cerr = w.abs() / D * (slope * (err + tol.U * (2 * diff + 2 * d + 16)) +
                          kl * (e + d + 1) * 8 * tol.U)
    lerr = (cerr + w.abs() / D * tol.U * 8 * (slope + adv.double().abs() * 2)).sum()
    return loss, lerr + tol.U * loss.abs(), lp, coef, cerr + 8 * tol.U * coef.abs(), keep, err


def _compare(x, labels, old, ref, adv, mask, kl, got, temperature=1.0, denom=None, gout=1.0):
    loss, logp, d = got
    v = x.shape[-1]
    want, lerr, lp, coef, cerr, keep, err = _expect(x, labels, old, ref, adv, mask, kl,
                                                    temperature, denom)
    assert abs(loss.item() - want.item()) <= lerr
    got_lp = logp.detach().cpu().double().reshape(-1)
    assert torch.all((got_lp - torch.where(keep, lp, 0.0)).abs() <= torch.where(keep, err, 0.0))
    flat, lab = x.reshape(-1, v), labels.reshape(-1)
    wd = orow.dlogits(flat, lab, coef * gout, temperature, keep)
    bound = tol.dlogits_error(flat, lab, coef * gout, cerr * abs(gout), wd, d.dtype, temperature)
    assert torch.all((d.cpu().double().reshape(-1, v) - wd).abs()
                     <= torch.where(keep[:, None], bound, 0.0))


def _run(x, labels, old, ref, adv, mask, kl, how, temperature=1.0, denom=None, gout=1.0):
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    c = lambda t: None if t is None else t.cuda()
    opts = dict(ref_logp=c(ref), mask=c(mask), clip_low=LOW, clip_high=HIGH, kl_coef=kl,
                temperature=temperature, denom=denom)
    xd = x.cuda()
    if how == "train":
        xd.requires_grad_(True)
        loss, logp = policy_loss(xd, c(labels), c(old), c(adv), **opts)
        assert not logp.requires_grad
        (d,) = torch.autograd.grad(loss * gout, xd)
        return loss.detach(), logp, d
    loss, logp, d = policy_loss_and_grad(xd, c(labels), c(old), c(adv), inplace=how == "inplace",
                                         **opts)
    assert x.numel() == 0 or (d.data_ptr() == xd.data_ptr()) == (how == "inplace")
    return loss, logp, d


# the fused kernel changes at 128, 512, 1024, 2048, 4096, 8192 and 16384 windows of 4 or 8
@pytest.mark.parametrize("how", ["step", "inplace", "train"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("v", [1, 3, 7, 8, 33, 511, 513, 2047, 2050, 4099, 8190, 16387, 32771,
                               65540, 131080])
def test_widths(v, dtype, how):
    announce(f"policy_loss width {v} {dtype} {how}")
    b, s = (3, 5) if v < 5000 else (2, 2)
    g, x, labels, old, ref, adv = _inputs(b, s, v, dtype)
    mask = torch.rand(b, s, generator=g) < 0.7
    mask[0, 0] = True
    labels[-1, -1] = orow.IGNORE
    got = _run(x, labels, old, ref, adv, mask, 0.05, how)
    _compare(x, labels, old, ref, adv, mask, 0.05, got)


@pytest.mark.parametrize("how", ["step", "train"])
@pytest.mark.parametrize("b,s", [(1, 1), (1, 700), (64, 3), (5, 1000)])
def test_batches(b, s, how):
    announce(f"policy_loss batch {b} x {s} {how}")
    g, x, labels, old, ref, adv = _inputs(b, s, 130, torch.float32, temperature=0.8)
    got = _run(x, labels, old, ref, adv, None, 0.02, how, temperature=0.8)
    _compare(x, labels, old, ref, adv, None, 0.02, got, temperature=0.8)


def test_weights_denominator_and_upstream_gradient():
    announce("policy_loss weights, denom, gout")
    g, x, labels, old, ref, adv = _inputs(4, 9, 77, torch.float32)
    w = torch.rand(4, 9, generator=g) * (torch.rand(4, 9, generator=g) < 0.8)
    got = _run(x, labels, old, None, adv, w, 0.0, "train", denom=5.0, gout=-3.0)
    _compare(x, labels, old, None, adv, w, 0.0, got, denom=5.0, gout=-3.0)
    got = _run(x, labels, old, None, adv, w, 0.0, "step")
    _compare(x, labels, old, None, adv, w, 0.0, got)


@pytest.mark.parametrize("shape", ["b", "b1", "scalar", "1s", "view"])
def test_advantages_broadcast(shape):
    announce(f"policy_loss advantages {shape}")
    g, x, labels, old, ref, adv = _inputs(3, 6, 50, torch.float32)
    if shape == "b":
        a, adv = adv[:, 0].contiguous(), adv[:, :1].expand(3, 6)
    elif shape == "b1":
        a, adv = adv[:, :1], adv[:, :1].expand(3, 6)
    elif shape == "scalar":
        a, adv = adv[0, 0], adv[0, 0].expand(3, 6)
    elif shape == "1s":
        a, adv = adv[:1], adv[:1].expand(3, 6)
    else:
        a = adv.T.contiguous().T
    got = _run(x, labels, old, ref, a, None, 0.1, "step")
    _compare(x, labels, old, ref, adv, None, 0.1, got)


def test_next_token_view_and_flat_rows():
    announce("policy_loss layouts")
    g, x, labels, old, ref, adv = _inputs(3, 6, 201, torch.bfloat16)
    from cases.policy_loss.op import policy_loss_and_grad
    wide = torch.cat([x, torch.full((3, 1, 201), float("nan"), dtype=x.dtype)], 1).cuda()
    got = policy_loss_and_grad(wide[:, :-1], labels.cuda(), old.cuda(), adv.cuda(),
                               clip_low=LOW, clip_high=HIGH)
    _compare(x, labels, old, None, adv, None, 0.0, got)
    flat = policy_loss_and_grad(x.cuda().view(18, 201), labels.cuda().view(18),
                                old.cuda().view(18), adv.cuda().view(18), clip_low=LOW,
                                clip_high=HIGH)
    assert all(torch.equal(p.reshape(-1), q.reshape(-1)) for p, q in zip(got, flat))


@pytest.mark.parametrize("how", ["step", "inplace", "train"])
@pytest.mark.parametrize("v", [40, 3000, 70000])
def test_masked_places_may_hold_anything(v, how):
    announce(f"policy_loss junk in masked places {v} {how}")
    g, x, labels, old, ref, adv = _inputs(3, 4, v, torch.float32)
    mask = torch.ones(3, 4, dtype=torch.bool)
    mask[1] = False                      # an answer without a token
    mask[2, 3] = False
    labels[0, 2] = orow.IGNORE
    clean = _run(x, labels, old, ref, adv, mask, 0.05, how, gout=2.0 if how == "train" else 1.0)
    _compare(x, labels, old, ref, adv, mask, 0.05, clean, gout=2.0 if how == "train" else 1.0)
    for t, junk in ((x, float("nan")), (old, float("inf")), (ref, float("nan")),
                    (adv, float("nan"))):
        t[~mask] = junk
        t[0, 2] = junk
    labels[1] = 10 ** 12
    dirty = _run(x, labels, old, ref, adv, mask, 0.05, how, gout=2.0 if how == "train" else 1.0)
    assert all(torch.equal(p, q) for p, q in zip(clean, dirty))


@pytest.mark.parametrize("how", ["step", "train"])
def test_nothing_counts(how):
    announce(f"policy_loss of nothing {how}")
    g, x, labels, old, ref, adv = _inputs(2, 3, 20, torch.float32)
    loss, logp, d = _run(x, labels, old, ref, adv, torch.zeros(2, 3, dtype=torch.bool), 0.1, how)
    assert loss.item() == 0 and not logp.any() and not d.any()
    e = torch.empty(0, 20), torch.empty(0, dtype=torch.int64), torch.empty(0)
    loss, logp, d = _run(e[0], e[1], e[2], None, e[2], None, 0.0, how)
    assert loss.item() == 0 and d.shape == (0, 20)


def test_label_outside_the_row_and_nan_logits():
    announce("policy_loss invalid labels")
    for how in ("step", "train"):
        g, x, labels, old, ref, adv = _inputs(1, 4, 600, torch.float32)
        labels[0, 1] = 600
        x[0, 2, 5] = float("nan")
        loss, logp, d = _run(x, labels, old, ref, adv, None, 0.1, how)
        assert torch.isnan(loss)
        assert torch.isnan(d[0, 1]).all() and torch.isnan(d[0, 2]).all()
        assert torch.isfinite(d[0, 0]).all() and torch.isfinite(d[0, 3]).all()


def test_gradient_against_differences():
    """Directional differences of the 64-bit loss against the kernels' gradient."""
    announce("policy_loss differences")
    g, x, labels, old, ref, adv = _inputs(2, 5, 30, torch.float32)
    _, _, d = _run(x, labels, old, ref, adv, None, 0.1, "step")

    def loss(y):
        lp = orow.logp(y.reshape(-1, 30), labels.reshape(-1))
        return orow.policy(lp, labels.reshape(-1), old.reshape(-1), adv.reshape(-1),
                           ref.reshape(-1), None, LOW, HIGH, 0.1)[0]
    h = 1e-5
    for i in range(4):
        e = torch.randn(x.shape, generator=g, dtype=torch.float64)
        diff = (loss(x.double() + h * e) - loss(x.double() - h * e)) / (2 * h)
        assert abs(diff - (d.cpu().double() * e).sum()) <= 1e-6 * e.norm()


def test_backward_twice_and_repeats():
    announce("policy_loss backward twice")
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    g, x, labels, old, ref, adv = _inputs(3, 50, 5000, torch.bfloat16)
    xd = x.cuda().requires_grad_(True)
    args = labels.cuda(), old.cuda(), adv.cuda(), ref.cuda()
    loss, _ = policy_loss(xd, *args, kl_coef=0.1)
    (a,) = torch.autograd.grad(loss, xd, retain_graph=True)
    (b,) = torch.autograd.grad(loss, xd)
    assert torch.equal(a, b)
    one, two = (policy_loss_and_grad(xd, *args, kl_coef=0.1) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    assert torch.equal(one[0], loss)


def test_graph_replays_on_new_inputs():
    announce("policy_loss captured")
    from cases.policy_loss.op import policy_loss_and_grad
    g, x, labels, old, ref, adv = _inputs(2, 20, 3000, torch.bfloat16)
    xd, args = x.cuda(), (labels.cuda(), old.cuda(), adv.cuda(), ref.cuda())
    policy_loss_and_grad(xd, *args, kl_coef=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = policy_loss_and_grad(xd, *args, kl_coef=0.1)
    for i in range(4):
        xd.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
        want = policy_loss_and_grad(xd, *args, kl_coef=0.1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_another_stream():
    announce("policy_loss on a side stream")
    from cases.policy_loss.op import policy_loss
    g, x, labels, old, ref, adv = _inputs(2, 20, 3000, torch.float32)
    xd = x.cuda().requires_grad_(True)
    args = labels.cuda(), old.cuda(), adv.cuda()
    (want,) = torch.autograd.grad(policy_loss(xd, *args)[0], xd)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        (got,) = torch.autograd.grad(policy_loss(xd, *args)[0], xd)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_more_than_2_to_the_31_logits():
    announce("policy_loss over 2^31 elements")
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    rows, v = 65536 + 4, 32776
    assert rows * v > 2 ** 31
    logits = torch.zeros(rows, v, dtype=torch.bfloat16, device="cuda")
    g, x, labels, old, ref, adv = _inputs(1, 4, v, torch.bfloat16)
    logits[-4:] = x[0].cuda()
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[-4:] = True
    full = [torch.zeros(rows, dtype=t.dtype, device="cuda") for t in (labels, old, adv)]
    for f, t in zip(full, (labels, old, adv)):
        f[-4:] = t[0].cuda()
    opts = dict(mask=mask, clip_low=LOW, clip_high=HIGH)
    loss, logp, d = policy_loss_and_grad(logits, *full, **opts)
    assert not d[:-4].any()
    _compare(x, labels, old, None, adv, None, 0.0, (loss, logp[-4:], d[-4:]))
    del d
    logits.requires_grad_(True)
    loss, logp = policy_loss(logits, *full, **opts)
    (d,) = torch.autograd.grad(loss, logits)
    assert not d[:-4].any()
    _compare(x, labels, old, None, adv, None, 0.0, (loss.detach(), logp[-4:], d[-4:]))


def test_refusals():
    announce("policy_loss refusals")
    from cases.policy_loss.op import policy_loss, policy_loss_and_grad
    g, x, labels, old, ref, adv = _inputs(2, 3, 20, torch.float32)
    x, labels, old, ref, adv = (t.cuda() for t in (x, labels, old, ref, adv))
    ok = (x, labels, old, adv)
    for kw in (dict(kl_coef=0.1), dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_high=-1.0),
               dict(clip_high=float("nan")), dict(temperature=0.0), dict(denom=0.0),
               dict(denom=-1.0), dict(denom=float("inf")), dict(kl_coef=-1.0, ref_logp=ref),
               dict(mask=torch.ones(2, 4, dtype=torch.bool, device="cuda")),
               dict(mask=torch.ones(2, 3, dtype=torch.int64, device="cuda")),
               dict(mask=torch.ones(2, 3, dtype=torch.bool)), dict(ref_logp=ref.double()),
               dict(ref_logp=ref.cpu())):
        with pytest.raises(RuntimeError):
            policy_loss(*ok, **kw)
        with pytest.raises(RuntimeError):
            policy_loss_and_grad(*ok, **kw)
    for bad in ((x, labels, old[:1, :2], adv), (x, labels, old, adv[:, :2]),
                (x, labels, old.bfloat16(), adv), (x, labels, old, adv.double())):
        with pytest.raises(RuntimeError):
            policy_loss(*bad)
    with pytest.raises(RuntimeError):
        policy_loss_and_grad(x[:, :-1], labels[:, :-1], old[:, :-1], adv[:, :-1], inplace=True)
