"""Matrices with a short side, whose steps run in 64 bits on the Gram matrix:
both sides of its limits, ranks that are not full, and the steps past which the
general way takes over.  Against the SVD oracle: a result is rounded once to
its type, and Q, of 2^-53 operands whose errors grow by a^2 a step, is off by
less than 1e9 * 2^-53 of its size."""

import pytest
import torch

from conftest import announce
from oracle import newton_schulz as ons

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _matrix(m, n, rank=None, dtype=torch.float32):
    g = torch.Generator().manual_seed(1000 * m + n)
    r = min(m, n) if rank is None else rank
    return (torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g)).to(dtype)


def _close(got, G, slack=1e-7, **ns):
    want = ons.orthogonalise(G, **ns)
    bound = (EPS[got.dtype] * 1.01 + slack) * want.abs() + slack * want.abs().max() + 2.0 ** -25
    assert torch.all((got.cpu().double() - want).abs() <= bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("l", [64, 65, 127, 1000, 5000])
def test_sides(k, l, dtype):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz short side {k} x {l} {dtype}")
    for m, n in ((k, l), (l, k)):
        G = _matrix(m, n, dtype=dtype)
        _close(newton_schulz(G.cuda()), G)


@pytest.mark.parametrize("rank", [1, 5, 39])
def test_ranks(rank):
    """Exact low rank: the directions outside it stay 0."""
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz short side, rank {rank}")
    g = torch.Generator().manual_seed(rank)
    G = (torch.randint(-4, 5, (40, rank), generator=g).float() @
         torch.randint(-4, 5, (rank, 300), generator=g).float())
    _close(newton_schulz(G.cuda()), G, slack=2e-6)


@pytest.mark.parametrize("steps", [1, 2, 8, 9, 20])
def test_steps_on_both_sides_of_the_limit(steps):
    """Up to 8 steps of the default coefficients on the Gram matrix, then on X."""
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz short side, {steps} steps")
    G = _matrix(48, 90, rank=20) + 0.01 * _matrix(48, 90)
    got = newton_schulz(G.cuda(), steps=steps)
    want = ons.orthogonalise(G, steps=steps)
    off = ons.by_products(G, steps=steps, operand=2.0 ** -21, product=2.0 ** -22, seed=1)
    assert (got.cpu().double() - want).norm() <= 4 * (off - want).norm() + 1e-6 * want.norm()


@pytest.mark.parametrize("m,n", [(20, 300), (300, 20)])
def test_update_in_place_and_batches(m, n):
    from cases.newton_schulz.op import muon_step
    announce(f"muon_step short side {m} x {n}")
    W = [_matrix(m, n).cuda() * 0.01 for _ in range(35)]
    G = [(_matrix(m, n) + i * 0.1).cuda() for i in range(35)]
    M = [torch.zeros(m, n, device="cuda") for _ in range(35)]
    before = [w.cpu() for w in W]
    for _ in range(2):
        muon_step(W, G, M, lr=0.1, momentum=0.9, weight_decay=0.1)
    for i in (0, 1, 31, 32, 34):
        w, mom = before[i], torch.zeros(m, n)
        for _ in range(2):
            w, mom = ons.muon(w, G[i].cpu(), mom, 0.1, 0.9, weight_decay=0.1)
        assert (W[i].cpu().double() - w).abs().max() <= 1e-6
        assert (M[i].cpu().double() - mom).abs().max() <= 4 * 2.0 ** -24 * mom.abs().max()


def test_captured():
    from cases.newton_schulz.op import newton_schulz
    announce("newton_schulz short side captured")
    G = _matrix(50, 700).cuda()
    newton_schulz(G)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = newton_schulz(G)
    for i in range(4):
        G.copy_(_matrix(50, 700) + i * _matrix(700, 50).T)
        want = newton_schulz(G)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("precision", ["half", "full"])
def test_shapes_together(precision):
    """Weights of many shapes in one call: products in launches of their own and shared ones,
    short sides beside long ones, more shapes and matrices than a launch takes."""
    from cases.newton_schulz.op import muon_step
    announce(f"muon_step of many shapes {precision}")
    shapes = ([(70, 130)] * 40 + [(130, 70)] * 3 + [(96, 96)] * 35 + [(200, 520)] * 2 +
              [(20, 90)] * 33 + [(65, 66)] + [(300, 100)] * 2 + [(64, 64)])
    g = torch.Generator().manual_seed(3)
    W = [torch.randn(s, generator=g) * 0.02 for s in shapes]
    G = [_matrix(*s) * (1 + 0.1 * i) + 0.1 * torch.randn(s, generator=g)
         for i, s in enumerate(shapes)]
    M = [0.3 * torch.randn(s, generator=g) for s in shapes]
    Wd, Gd, Md = ([t.cuda() for t in x] for x in (W, G, M))
    muon_step(Wd, Gd, Md, lr=0.05, momentum=0.9, precision=precision)
    again = [w.cuda() for w in W]
    muon_step(again, Gd, [m.cuda() for m in M], lr=0.05, momentum=0.9, precision=precision)
    assert all(torch.equal(a, b) for a, b in zip(Wd, again))
    size = {"half": 2.0 ** -11, "full": 2.0 ** -21}[precision]
    for i in range(0, len(shapes), 3):
        U = G[i].double() + 0.9 * (0.9 * M[i].double() + G[i].double())
        s = max(1.0, shapes[i][0] / shapes[i][1]) ** 0.5
        O = ons.orthogonalise(U)
        off = ons.by_products(U, operand=size, product=2.0 ** -22, seed=1)
        want = W[i].double() - 0.05 * s * O
        bound = 0.05 * s * 4 * (off - O).norm() + 2.0 ** -22 * (want.norm() + O.norm())
        assert (Wd[i].cpu().double() - want).norm() <= bound, shapes[i]
