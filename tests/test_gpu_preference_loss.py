"""The preference loss on the GPU, padded and packed, against the float64
oracle.  A sequence's sum is off by the sum of its tokens' logp errors
(operator_tolerances.py) and a rounding; a pair's coefficient by a quarter of
beta times the difference's error (the logistic function's steepest slope)."""

import pytest
import torch

import operator_tolerances as tol
from conftest import announce
from oracle import token_rows as orow

pytestmark = pytest.mark.gpu


def _rows(n2, lens, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    total = sum(lens)
    x = (torch.randn(total, v, generator=g) * 2).to(dtype)
    labels = torch.randint(0, v, (total,), generator=g)
    seqs, at = [], 0
    for n in lens:
        seqs.append(torch.arange(at, at + n))
        if n > 2:
            labels[at] = orow.IGNORE       # a prompt
        at += n
    ref = torch.stack([orow.logp(x[s], labels[s]).sum() for s in seqs]).float()
    return g, x, labels, seqs, ref + torch.randn(n2, generator=g)


def _compare(x, labels, seqs, ref, got, beta, eps, average, gout=1.0):
    loss, seq, d = got
    lp = orow.logp(x, labels)
    want, wseq, coef = orow.preference(lp, labels, seqs, ref, beta, eps, average)
    keep = labels != orow.IGNORE
    err = torch.where(keep, tol.logp_error(x, labels, lp), 0.0)
    share = torch.tensor([1.0 / max(1, int(keep[s].sum())) if average else 1.0 for s in seqs],
                         dtype=torch.float64)
    serr = torch.stack([err[s].sum() for s in seqs]) * share
    assert torch.all((seq.cpu().double() - wseq).abs() <= serr + 2 * tol.U * wseq.abs() + 1e-300)
    n = len(seqs) // 2
    derr = abs(beta) * (serr[:n] + serr[n:]) + 1e-12
    assert abs(loss.item() - want) <= derr.mean() + 4 * tol.U * want.abs()
    cerr = torch.zeros_like(lp)
    for i in range(2 * n):
        size = abs(beta) / n * share[i] * derr[i % n] / 4
        cerr[seqs[i]] = size + 6 * tol.U * coef[seqs[i]].abs()
    wd = orow.dlogits(x, labels, coef * gout)
    bound = tol.dlogits_error(x, labels, coef * gout, cerr * abs(gout), wd, d.dtype)
    live = keep & (coef != 0)
    assert torch.all((d.cpu().double() - wd).abs() <= torch.where(live[:, None], bound, 0.0))


def _run(x, labels, ref, how, cu=None, gout=1.0, **opts):
    from cases.preference_loss.op import preference_loss, preference_loss_and_grad
    args = labels.cuda(), None if ref is None else ref.cuda()
    cu = None if cu is None else cu.cuda()
    xd = x.cuda()
    if how == "step":
        return preference_loss_and_grad(xd, *args, cu_seqlens=cu, **opts)
    xd.requires_grad_(True)
    loss, seq = preference_loss(xd, *args, cu_seqlens=cu, **opts)
    assert not seq.requires_grad
    (d,) = torch.autograd.grad(loss * gout, xd)
    return loss.detach(), seq, d


LENGTHS = [(5, 1, 3, 9), (1, 1), (0, 7), (300, 2, 257, 64, 0, 1)]


@pytest.mark.parametrize("how", ["step", "train"])
@pytest.mark.parametrize("average,eps", [(False, 0.0), (True, 0.1)])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_packed(lens, average, eps, how):
    announce(f"preference_loss packed {lens} average={average} {how}")
    g, x, labels, seqs, ref = _rows(len(lens), lens, 203, torch.float32, 11)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)))
    gout = -2.0 if how == "train" else 1.0
    got = _run(x, labels, ref, how, cu, gout, beta=0.3, label_smoothing=eps, average=average)
    _compare(x, labels, seqs, ref, got, 0.3, eps, average, gout)


@pytest.mark.parametrize("how", ["step", "train"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,s,v", [(1, 1, 1), (2, 7, 50), (1, 300, 1001), (5, 3, 9000),
                                   (1, 2, 70001)])
def test_padded(n, s, v, dtype, how):
    announce(f"preference_loss {n} pairs x {s} x {v} {dtype} {how}")
    g, x, labels, seqs, ref = _rows(2 * n, [s] * 2 * n, v, dtype, 5)
    if s > 3:
        labels.view(2 * n, s)[1, s // 2:] = orow.IGNORE
    got = _run(x.view(2 * n, s, v), labels.view(2 * n, s), ref, how, beta=0.2)
    got = got[0], got[1], got[2].reshape(-1, v)
    _compare(x, labels, seqs, ref, got, 0.2, 0.0, False)


def test_padded_and_packed_agree():
    announce("preference_loss padded against packed")
    g, x, labels, seqs, ref = _rows(4, [20] * 4, 333, torch.bfloat16, 6)
    a = _run(x.view(4, 20, 333), labels.view(4, 20), ref, "step", average=True)
    b = _run(x, labels, ref, "step", torch.arange(0, 81, 20), average=True)
    assert all(torch.equal(p.reshape(-1), q.reshape(-1)) for p, q in zip(a, b))


def test_rows_in_no_sequence_and_offsets_outside():
    """Rows before the first and after the last offset get zeros; offsets past the rows end
    there, and ones that run backwards make an empty sequence."""
    announce("preference_loss offsets")
    g, x, labels, seqs, ref = _rows(2, [10, 10], 40, torch.float32, 7)
    loss, seq, d = _run(x, labels, ref, "step", torch.tensor([3, 9, 15]))
    assert not d[:3].any() and not d[15:].any() and d[4:15].any()
    _compare(x, labels, [torch.arange(3, 9), torch.arange(9, 15)], ref, (loss, seq, d), 0.1, 0.0,
             False)
    loss, seq, d = _run(x, labels, ref, "step", torch.tensor([-5, 10, 1 << 40]))
    _compare(x, labels, [torch.arange(0, 10), torch.arange(10, 20)], ref, (loss, seq, d), 0.1, 0.0,
             False)
    loss, seq, d = _run(x, labels, ref, "step", torch.tensor([10, 4, 20]))
    assert seq[0] == 0 and torch.isfinite(loss)


def test_far_apart_pairs_stay_finite():
    announce("preference_loss large differences")
    g, x, labels, seqs, _ = _rows(4, [6] * 4, 30, torch.float32, 8)
    for size in (300.0, -300.0):
        ref = torch.tensor([size, 0.0, 0.0, 0.0])
        got = _run(x.view(4, 6, 30), labels.view(4, 6), ref, "step", beta=1.0)
        got = got[0], got[1], got[2].reshape(-1, 30)
        _compare(x, labels, seqs, ref, got, 1.0, 0.0, False)
    without = _run(x.view(4, 6, 30), labels.view(4, 6), None, "step")
    _compare(x, labels, seqs, torch.zeros(4), (without[0], without[1],
                                               without[2].reshape(-1, 30)), 0.1, 0.0, False)


def test_gradient_against_differences():
    announce("preference_loss differences")
    g, x, labels, seqs, ref = _rows(4, [5, 3, 4, 6], 25, torch.float32, 9)
    _, _, d = _run(x, labels, ref, "step", torch.tensor([0, 5, 8, 12, 18]), beta=0.5,
                   label_smoothing=0.1)

    def loss(y):
        return orow.preference(orow.logp(y, labels), labels, seqs, ref, 0.5, 0.1)[0]
    h = 1e-5
    for _ in range(4):
        e = torch.randn(x.shape, generator=g, dtype=torch.float64)
        diff = (loss(x.double() + h * e) - loss(x.double() - h * e)) / (2 * h)
        assert abs(diff - (d.cpu().double() * e).sum()) <= 1e-6 * e.norm()


def test_ignored_rows_may_hold_anything_and_repeats():
    announce("preference_loss junk in ignored places")
    g, x, labels, seqs, ref = _rows(2, [8, 8], 500, torch.bfloat16, 10)
    a = _run(x.view(2, 8, 500), labels.view(2, 8), ref, "step")
    x[labels == orow.IGNORE] = float("nan")
    b = _run(x.view(2, 8, 500), labels.view(2, 8), ref, "step")
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graph_replays_on_new_inputs():
    announce("preference_loss captured")
    from cases.preference_loss.op import preference_loss_and_grad
    g, x, labels, seqs, ref = _rows(4, [9] * 4, 700, torch.float32, 12)
    xd, ld, rd = x.view(4, 9, 700).cuda(), labels.view(4, 9).cuda(), ref.cuda()
    preference_loss_and_grad(xd, ld, rd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = preference_loss_and_grad(xd, ld, rd)
    for _ in range(4):
        xd.copy_(torch.randn(xd.shape, generator=g))
        want = preference_loss_and_grad(xd, ld, rd)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals():
    announce("preference_loss refusals")
    from cases.preference_loss.op import preference_loss
    x = torch.zeros(4, 3, 8, device="cuda")
    l = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    cu = torch.tensor([0, 6, 12], device="cuda")
    for bad in (lambda: preference_loss(x[:3], l[:3]), lambda: preference_loss(x[0], l[0]),
                lambda: preference_loss(x, l, torch.zeros(3, device="cuda")),
                lambda: preference_loss(x, l, torch.zeros(4, device="cuda").double()),
                lambda: preference_loss(x, l, cu_seqlens=cu),
                lambda: preference_loss(x.view(12, 8), l.view(12), cu_seqlens=cu.int()),
                lambda: preference_loss(x.view(12, 8), l.view(12), cu_seqlens=cu[:2]),
                lambda: preference_loss(x.view(12, 8), l.view(12), cu_seqlens=cu.cpu()),
                lambda: preference_loss(x, l, label_smoothing=1.5),
                lambda: preference_loss(x, l, beta=float("inf")),
                lambda: preference_loss(x.double(), l), lambda: preference_loss(x, l.int())):
        with pytest.raises(RuntimeError):
            bad()
