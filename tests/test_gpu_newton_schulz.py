"""Newton-Schulz updates on the GPU against the float64 oracle (an SVD).

How far off a result may be is taken from the oracle itself: the same iteration
in 64 bits with its operands and products off by random roundings of the
kernels' sizes lies some distance from the exact one, and the kernels' result
must lie within four of those, and within the rounding to its own type.
Operands: 2^-11 a half (to nearest, 2^-12, and a bit for float16's scale), 2^-21
a full one.  Products: 32-bit sums, 2^-22 of the sum of their terms' sizes."""

import pytest
import torch

from conftest import announce
from oracle import newton_schulz as ons

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
OPERAND = {"half": 2.0 ** -11, "full": 2.0 ** -21}
PRODUCT = 2.0 ** -22


def _matrix(m, n, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + 1000 * m + n)
    r = max(1, min(m, n) // 4)
    x = torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) / r ** 0.5
    return ((x + 0.3 * torch.randn(m, n, generator=g)) * 1e-3).to(dtype)


def _default(dtype):
    return "full" if dtype == torch.float32 else "half"


def _close(got, G, precision, dtype=None, factor=1.0, **ns):
    """got = factor * the orthogonalised G."""
    want = ons.orthogonalise(G, **ns)
    off = ons.by_products(G, operand=OPERAND[precision], product=PRODUCT, seed=1, **ns)
    bound = 4 * (off - want).norm() + 1e-300
    bound = bound + EPS[dtype or got.dtype] * want.norm() * 1.01
    assert (got.cpu().double() / factor - want).norm() <= bound


SHAPES = [(1, 1), (1, 9), (9, 1), (7, 3), (16, 16), (31, 33), (32, 64), (64, 64), (65, 63),
          (100, 31), (128, 128), (130, 257), (257, 130), (300, 1000), (513, 511)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(m, n, dtype):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz {m} x {n} {dtype}")
    G = _matrix(m, n, dtype=dtype)
    out = newton_schulz(G.cuda())
    assert out.dtype == dtype and out.shape == G.shape
    _close(out, G, _default(dtype))


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_precision_asked_for(dtype, precision):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz precision {precision} {dtype}")
    G = _matrix(150, 200, dtype=dtype)
    _close(newton_schulz(G.cuda(), precision=precision), G, precision)


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("m,n", [(1100, 1300), (2000, 600)])
def test_large(m, n, precision):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz {m} x {n} {precision}")
    G = torch.stack([_matrix(m, n, s) for s in range(3)])
    out = newton_schulz(G.cuda(), precision=precision)
    for i in range(3):
        _close(out[i], G[i], precision)


@pytest.mark.parametrize("count", [1, 3, 32, 33, 70])
def test_batches(count):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz {count} matrices")
    G = torch.stack([_matrix(20, 45, s) for s in range(count)])
    out = newton_schulz(G.cuda())
    for i in range(count):
        _close(out[i], G[i], "full")
    alone = newton_schulz(G[count // 2].cuda())
    assert torch.equal(alone, out[count // 2])


@pytest.mark.parametrize("layout", ["rows_apart", "offset", "transposed", "batch_strided", "four",
                                    "expanded", "columns"])
def test_layouts(layout):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz layout {layout}")
    base = _matrix(80, 91)
    if layout == "rows_apart":
        G = base.cuda()[:, 3:70]
    elif layout == "offset":
        G = base.cuda().flatten()[1:1 + 60 * 91].view(60, 91)
    elif layout == "transposed":
        G = base.cuda().T
    elif layout == "batch_strided":
        G = base.cuda().view(4, 20, 91)[::2, 3:17]
    elif layout == "four":
        G = base.cuda().view(2, 2, 20, 91)
    elif layout == "columns":
        G = base.cuda()[:, ::3]
    else:
        G = base.cuda()[:1].expand(40, 91)
    out = newton_schulz(G)
    assert out.shape == G.shape
    flat, of = G.cpu().reshape(-1, *G.shape[-2:]), out.reshape(-1, *G.shape[-2:])
    for i in range(flat.shape[0]):
        _close(of[i], flat[i], "full")


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e18, 3e30])
def test_sizes_of_elements(size):
    """Squares that leave 32 bits on either side; eps counts where the norm is as small."""
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz elements of {size}")
    G = _matrix(40, 50) * 1e3 * size
    _close(newton_schulz(G.cuda(), eps=0.0), G, "full", eps=0.0)
    if size >= 1e-6:
        _close(newton_schulz(G.cuda()), G, "full")


def test_zeros_nan_and_empty():
    from cases.newton_schulz.op import newton_schulz
    announce("newton_schulz zeros, NaN, empty")
    G = torch.stack([_matrix(30, 40), torch.zeros(30, 40), _matrix(30, 40, 2), _matrix(30, 40, 3)])
    G[2, 3, 4] = float("nan")
    G[3, 0, 0] = float("inf")
    for eps in (1e-7, 0.0):
        out = newton_schulz(G.cuda(), eps=eps).cpu()
        _close(out[0], G[0], "full", eps=eps)
        assert not out[1].any()
        assert torch.isnan(out[2]).all() and torch.isnan(out[3]).all()
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 4)):
        assert newton_schulz(torch.empty(shape, device="cuda")).shape == shape


@pytest.mark.parametrize("coefficients,steps", [((3.4445, -4.7750, 2.0315), 1),
                                                ((3.4445, -4.7750, 2.0315), 8),
                                                ((1.5, -0.5, 0.0), 12),
                                                ((1.875, -1.25, 0.375), 6), ((0.5, 0.0, 0.0), 2)])
def test_coefficients(coefficients, steps):
    from cases.newton_schulz.op import newton_schulz
    announce(f"newton_schulz {coefficients} x {steps}")
    G = _matrix(70, 90)
    _close(newton_schulz(G.cuda(), steps=steps, coefficients=coefficients), G, "full",
           steps=steps, coefficients=coefficients)


def test_graph_replays_and_repeats():
    from cases.newton_schulz.op import newton_schulz
    announce("newton_schulz captured")
    G = torch.stack([_matrix(100, 140, s) for s in range(2)]).cuda()
    newton_schulz(G)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = newton_schulz(G)
    for s in range(4):
        G.copy_(torch.stack([_matrix(100, 140, 10 + s + i) for i in range(2)]))
        want = newton_schulz(G)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_another_stream():
    from cases.newton_schulz.op import newton_schulz
    announce("newton_schulz on a side stream")
    G = _matrix(200, 300).cuda()
    want = newton_schulz(G)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = newton_schulz(G)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("nesterov,decay,scale", [(True, 0.0, None), (False, 0.1, 0.3)])
@pytest.mark.parametrize("wt,gt,mt", [(torch.float32, torch.float32, torch.float32),
                                      (torch.float32, torch.bfloat16, torch.float32),
                                      (torch.bfloat16, torch.bfloat16, torch.float32),
                                      (torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                      (torch.float16, torch.float32, torch.float16)], ids=str)
def test_muon_step(wt, gt, mt, nesterov, decay, scale):
    from cases.newton_schulz.op import muon_step
    announce(f"muon_step {wt} {gt} {mt} nesterov={nesterov}")
    g = torch.Generator().manual_seed(2)
    shapes = [(40, 70), (70, 40), (40, 70), (33, 33)]
    W = [(torch.randn(s, generator=g) * 0.02).to(wt) for s in shapes]
    G = [_matrix(*s, seed=i, dtype=gt) for i, s in enumerate(shapes)]
    M = [(0.5 * _matrix(*s, seed=9 + i)).to(mt) for i, s in enumerate(shapes)]
    Wd, Gd, Md = ([t.cuda() for t in x] for x in (W, G, M))
    muon_step(Wd, Gd, Md, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay,
              scale=scale)
    for w, x, mom, wd, md in zip(W, G, M, Wd, Md):
        kept = 0.9 * mom.double() + x.double()
        # mu in 32 bits and one rounding of the sum; then that to the momentum's type
        size = 0.9 * mom.double().abs() + x.double().abs()
        tiny = 2.0 ** -25 if mt == torch.float16 else 0.0
        assert torch.all((md.cpu().double() - kept).abs()
                         <= EPS[mt] * kept.abs() * 1.01 + 2.0 ** -23 * size + tiny)
        kept = md.cpu().double()            # U is taken from the momentum as it is kept
        U = x.double() + 0.9 * kept if nesterov else kept
        s = max(1.0, w.shape[0] / w.shape[1]) ** 0.5 if scale is None else scale
        base = (1 - 0.05 * decay) * w.double()
        O = ons.orthogonalise(U)
        off = ons.by_products(U, operand=OPERAND[_default(wt)], product=PRODUCT, seed=1)
        want = base - 0.05 * s * O
        bound = 0.05 * s * 4 * (off - O).norm() + 2 * EPS[wt] * want.norm() + 2.0 ** -23 * (
            base.norm() + 0.05 * s * O.norm())
        assert (wd.cpu().double() - want).norm() <= bound


def test_muon_optimiser_on_views():
    """Weights that are rows of a larger buffer; what lies between stays as it was."""
    from cases.newton_schulz.op import Muon
    announce("Muon on strided weights")
    buf = torch.randn(50, 100, generator=torch.Generator().manual_seed(1)).cuda()
    before = buf.clone()
    p = torch.nn.Parameter(buf[:, :60])
    assert p.data_ptr() == buf.data_ptr()
    opt = Muon([p], lr=0.1, momentum=0.5)
    x = _matrix(50, 60).cuda()
    M = torch.zeros(50, 60)
    want = before[:, :60].cpu()
    for _ in range(3):
        p.grad = x.clone()
        opt.step()
        want, M = ons.muon(want, x.cpu(), M, 0.1, 0.5)
    assert (p.detach().cpu().double() - want).abs().max() <= 1e-5
    assert torch.equal(buf[:, 60:], before[:, 60:])
    with pytest.raises(RuntimeError):
        Muon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])


def test_refusals():
    from cases.newton_schulz.op import muon_step, newton_schulz
    announce("newton_schulz refusals")
    G = torch.randn(4, 5, device="cuda")
    for bad in (lambda: newton_schulz(G.cpu()), lambda: newton_schulz(G.double()),
                lambda: newton_schulz(G[0]), lambda: newton_schulz(G, steps=0),
                lambda: newton_schulz(G, steps=1000), lambda: newton_schulz(G, eps=-1.0),
                lambda: newton_schulz(G, eps=float("nan")),
                lambda: newton_schulz(G, precision="low"),
                lambda: newton_schulz(G, coefficients=(9.0, 0.0, 0.0)),
                lambda: newton_schulz(G, coefficients=(float("nan"), 0.0, 0.0)),
                lambda: muon_step(G, G, G[:3], lr=0.1), lambda: muon_step([G], [G], [], lr=0.1),
                lambda: muon_step(G, G.cpu(), G, lr=0.1),
                lambda: muon_step(G.T, G.T, G.T, lr=0.1),
                lambda: muon_step(G, G, G.clone(), lr=float("inf"))):
        with pytest.raises(RuntimeError):
            bad()
