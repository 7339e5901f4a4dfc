"""Root-mean-square norm on the GPU against the float64 oracle: widths around every
kernel's edges, types of x, residual and weight, layouts, gradients, and the output
in 8 bits.  Bounds: layer_tolerances.py."""

import pytest
import torch

import layer_tolerances as tol
from conftest import announce
from oracle import layers as ol

pytestmark = pytest.mark.gpu

# the kernels change at 512, 1024, 2048, 4096, 8192, 16384 and 32768
WIDTHS = [1, 2, 7, 8, 9, 64, 127, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4100, 8192, 8193,
          16384, 16385, 32768, 32769, 40003]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# x, residual (None: without), weight
KINDS = [(torch.float32, None, torch.float32), (torch.float32, torch.float32, torch.bfloat16),
         (torch.bfloat16, None, torch.bfloat16), (torch.bfloat16, torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.float32, torch.bfloat16), (torch.float16, torch.float16, torch.float16),
         (torch.float16, torch.float32, torch.float32)]
EPS = 1e-5


def _inputs(rows, d, kind, seed=0):
    g = torch.Generator().manual_seed(seed + rows + d)
    x = torch.randn(rows, d, generator=g).to(kind[0])
    res = None if kind[1] is None else (2 * torch.randn(rows, d, generator=g)).to(kind[1])
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(kind[2])
    dy = (torch.randn(rows, d, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(kind[0])
    dh = None if kind[1] is None else torch.randn(rows, d, generator=g).to(kind[1])
    return x, res, w, dy, dh


def _gpu(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _check_forward(x, res, w, y, h):
    want, wh, r = ol.norm(x, w, res, EPS)
    assert y.dtype == x.dtype
    assert torch.all((y.cpu().double() - want).abs() <= tol.y_error(want, x.dtype))
    if res is not None:
        assert h.dtype == res.dtype and torch.equal(h.cpu().double(), wh)
    return want, wh, r


def _check_backward(x, res, w, dy, dh, wh, r, dx, dres, dw):
    want, wdw = ol.norm_backward(dy, wh, w, r, dh)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    err = (dx.cpu().double() - want).abs()
    assert torch.all(err <= tol.dx_error(dy, wh, w, r, dh, want, x.dtype))
    if res is not None:
        assert dres.dtype == res.dtype
        err = (dres.cpu().double() - want).abs()
        assert torch.all(err <= tol.dx_error(dy, wh, w, r, dh, want, res.dtype))
    err = (dw.cpu().double() - wdw).abs()
    assert torch.all(err <= tol.dw_error(dy, wh, r, wdw, w.dtype))


def _run(x, res, w, dy, dh):
    from cases.rms_norm.op import rms_norm
    xd, rd, wd, dyd, dhd = _gpu(x, res, w, dy, dh)
    for t in (xd, rd, wd):
        if t is not None:
            t.requires_grad_(True)
    if res is None:
        y, h, rest = rms_norm(xd, wd, eps=EPS), None, ()
        dx, dw = torch.autograd.grad(y, (xd, wd), dyd)
        dres = None
    else:
        y, h = rms_norm(xd, wd, rd, eps=EPS)
        dx, dres, dw = torch.autograd.grad((y, h), (xd, rd, wd), (dyd, dhd))
    with torch.no_grad():
        again = rms_norm(xd, wd, rd, eps=EPS)
        assert torch.equal(again if res is None else again[0], y)
    return y.detach(), h, dx, dres, dw


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: "-".join(str(t)[6:] for t in k))
@pytest.mark.parametrize("d", WIDTHS)
def test_widths(d, kind):
    rows = 9 if d < 5000 else 3
    announce(f"rms_norm {rows} x {d} {kind}")
    x, res, w, dy, dh = _inputs(rows, d, kind)
    y, h, dx, dres, dw = _run(x, res, w, dy, dh)
    _, wh, r = _check_forward(x, res, w, y, h)
    _check_backward(x, res, w, dy, dh, wh, r, dx, dres, dw)


@pytest.mark.parametrize("rows,d", [(1, 300), (2, 5000), (3000, 72), (2100, 700), (1500, 1500),
                                    (600, 9000), (300, 17000)])
def test_many_rows(rows, d):
    """On both sides of where a workgroup of the backward takes more than one."""
    announce(f"rms_norm {rows} x {d}")
    kind = (torch.bfloat16, torch.bfloat16, torch.float32)
    x, res, w, dy, dh = _inputs(rows, d, kind)
    y, h, dx, dres, dw = _run(x, res, w, dy, dh)
    _, wh, r = _check_forward(x, res, w, y, h)
    _check_backward(x, res, w, dy, dh, wh, r, dx, dres, dw)


def test_gradients_against_differences():
    """Of sum(dy y) + sum(dh h) in 32 bits: the third derivative's share of a step of 2^-6 and the
    values' roundings over it bound what a central difference may be off."""
    from cases.rms_norm.op import rms_norm
    announce("rms_norm differences")
    x, res, w, dy, dh = _inputs(2, 40, (torch.float32,) * 3)
    xd, rd, wd, dyd, dhd = _gpu(x, res, w, dy, dh)
    _, _, dx, _, dw = _run(x, res, w, dy, dh)

    def value(x, w):
        with torch.no_grad():
            y, h = rms_norm(x, w, rd, eps=EPS)
        return (y.double() * dyd).sum() + (h.double() * dhd).sum()
    step = 2.0 ** -6
    size = (dy.abs().sum() * 4 + dh.abs().sum() * 8).item()
    bound = 8 * size * step ** 2 + 16 * tol.U * size * 8 / step
    for i in range(0, 40, 3):
        e = torch.zeros_like(xd)
        e[1, i] = step
        d = (value(xd + e, wd) - value(xd - e, wd)) / (2 * step)
        assert abs(d - dx[1, i]) <= bound
        e = torch.zeros_like(wd)
        e[i] = step
        d = (value(xd, wd + e) - value(xd, wd - e)) / (2 * step)
        assert abs(d - dw[i]) <= bound


@pytest.mark.parametrize("which", ["y", "h", "weight_frozen", "x_frozen"])
def test_some_of_the_gradients(which):
    from cases.rms_norm.op import rms_norm
    announce(f"rms_norm gradient of {which}")
    x, res, w, dy, dh = _inputs(5, 300, (torch.bfloat16, torch.float32, torch.float32))
    xd, rd, wd, dyd, dhd = _gpu(x, res, w, dy, dh)
    leaves = {"weight_frozen": (xd, rd), "x_frozen": (wd,)}.get(which, (xd, rd, wd))
    for t in leaves:
        t.requires_grad_(True)
    y, h = rms_norm(xd, wd, rd, eps=EPS)
    _, wh, r = ol.norm(x, w, res, EPS)
    if which == "y":
        dh = None
        got = torch.autograd.grad(y, leaves, dyd)
    elif which == "h":
        dy = torch.zeros_like(dy)
        got = torch.autograd.grad(h, leaves, dhd)
        assert torch.equal(got[1], dhd) and torch.all(got[2] == 0)
    else:
        got = torch.autograd.grad((y, h) if which == "weight_frozen" else y, leaves,
                                  (dyd, dhd) if which == "weight_frozen" else dyd)
    want, wdw = ol.norm_backward(dy, wh, w, r, dh)
    by = {id(t): g for t, g in zip(leaves, got)}
    if id(xd) in by:
        assert torch.all((by[id(xd)].cpu().double() - want).abs() <=
                         tol.dx_error(dy, wh, w, r, dh, want, torch.bfloat16))
    if id(wd) in by:
        assert torch.all((by[id(wd)].cpu().double() - wdw).abs() <=
                         tol.dw_error(dy, wh, r, wdw, torch.float32))


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu], ids=str)
@pytest.mark.parametrize("kind", KINDS, ids=lambda k: "-".join(str(t)[6:] for t in k))
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 130), (2, 700), (17, 1111), (1, 4096), (130, 5000),
                                    (2, 16400), (2, 33000)])
def test_output_in_8_bits(rows, d, kind, scale_dtype):
    """Scales within the norm's own error of the oracle's, or the power of two on the other side of
    a border; codes within half a step and that error of the exact quotient."""
    from cases.rms_norm.op import rms_norm_quantized
    announce(f"rms_norm_quantized {rows} x {d} {kind} {scale_dtype}")
    x, res, w, _, _ = _inputs(rows, d, kind)
    xd, rd, wd = _gpu(x, res, w)
    codes, scales, *h = rms_norm_quantized(xd, wd, rd, eps=EPS, scale_dtype=scale_dtype)
    want, wh, _ = ol.norm(x, w, res, EPS)
    if res is not None:
        assert torch.equal(h[0].cpu().double(), wh)
    else:
        assert not h
    rel = tol.U * ((tol.adds(d) + 2) / 2 + 6)
    pad = torch.nn.functional.pad(want.abs(), (0, -d % 128)).view(rows, -1, 128).amax(-1)
    s = scales.cpu().float().double()
    assert s.shape == pad.shape
    if scale_dtype == torch.float32:
        assert torch.all((s - pad / 448).abs() <= pad / 448 * (rel + 2 * tol.U) + 2.0 ** -126)
    else:
        assert torch.all(torch.frexp(s)[0] == 0.5)
        assert torch.all(s * 448 >= pad * (1 - rel))
        assert torch.all((s * 224 < pad * (1 + rel)) | (s == 2.0 ** -126))
    each = ol.spread(s, rows, d)
    exact = want / each
    half = torch.maximum(exact.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64))
    got = codes.cpu().float().double()
    assert torch.all((got - exact).abs() <= (half + exact.abs() * rel) * (1 + 2.0 ** -20))
    p = -(-d // 16) * 16
    whole = codes.as_strided((rows, p), (p, 1)).view(torch.uint8)
    assert torch.all(whole[:, d:] == 0)


@pytest.mark.parametrize("layout", ["columns", "rows_apart", "offset", "expanded", "three", "vector",
                                    "transposed"])
def test_layouts(layout):
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce(f"rms_norm layout {layout}")
    g = torch.Generator().manual_seed(5)
    base = torch.randn(30, 900, generator=g).bfloat16().cuda()

    def view(b):
        return {"columns": b[:, ::2], "rows_apart": b[::3, 5:305],
                "offset": b.view(-1)[1:3001].view(10, 300), "expanded": b[:1].expand(20, 900),
                "three": b.view(3, 10, 900), "vector": b[3], "transposed": b.t()}[layout]
    x, res = view(base), view(base.flip(0).contiguous())
    w = torch.randn(x.size(-1), generator=g).bfloat16().cuda()
    leaf, rl, wl = (t.detach().requires_grad_(True) for t in (x, res, w))
    y, h = rms_norm(leaf, wl, rl, eps=EPS)
    dy = torch.randn(x.shape, generator=g).bfloat16()
    dx, dres, dw = torch.autograd.grad(y, (leaf, rl, wl), dy.cuda())
    flat = [t.cpu().reshape(-1, x.size(-1)) for t in (x, res, dy)]
    _, wh, r = _check_forward(flat[0], flat[1], w.cpu(), y.detach().reshape(-1, x.size(-1)),
                              h.detach().reshape(-1, x.size(-1)))
    assert y.shape == h.shape == dx.shape == x.shape
    _check_backward(flat[0], flat[1], w.cpu(), flat[2], None, wh, r,
                    *(t.reshape(-1, x.size(-1)) for t in (dx, dres)), dw)
    with torch.no_grad():
        codes, scales, h2 = rms_norm_quantized(x, w, res, eps=EPS)
    assert torch.equal(h2, h) and codes.shape == x.shape
    assert scales.shape == (*x.shape[:-1], -(-x.size(-1) // 128))


def test_upstream_gradients_of_other_layouts():
    """Expanded, transposed and sliced gradients."""
    from cases.rms_norm.op import rms_norm
    announce("rms_norm upstream layouts")
    x, res, w, dy, dh = _inputs(12, 40, (torch.float32,) * 3)
    xd, rd, wd = _gpu(x, res, w)
    for t in (xd, rd, wd):
        t.requires_grad_(True)
    y, h = rms_norm(xd, wd, rd, eps=EPS)
    for gy, gh in ((torch.ones((), device="cuda").expand(12, 40), dh.cuda().t().contiguous().t()),
                   (torch.randn(12, 80).cuda()[:, ::2], torch.randn(24, 40).cuda()[::2])):
        got = torch.autograd.grad((y, h), (xd, rd, wd), (gy, gh), retain_graph=True)
        want = torch.autograd.grad((y, h), (xd, rd, wd), (gy.contiguous(), gh.contiguous()),
                                   retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shared_and_broadcast_inputs():
    """The same tensor as x and residual; a row and a weight that are used more than once."""
    from cases.rms_norm.op import rms_norm
    announce("rms_norm shared inputs")
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 50, generator=g).cuda().requires_grad_(True)
    w = torch.randn(50, generator=g).cuda().requires_grad_(True)
    y, h = rms_norm(x, w, x, eps=EPS)
    z = rms_norm(h, w, eps=EPS)
    dx, dw = torch.autograd.grad(z.sum() + y.sum(), (x, w))
    xx, ww = (t.detach().cpu().double().requires_grad_(True) for t in (x, w))

    def plain(h):
        return h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * ww
    ex, ew = torch.autograd.grad(plain(2 * xx).sum() * 2, (xx, ww))
    assert torch.all((dx.cpu() - ex).abs() <= 1000 * tol.U * 50)
    assert torch.all((dw.cpu() - ew).abs() <= 1000 * tol.U * 8)
    row = torch.randn(1, 50, generator=g).cuda().requires_grad_(True)
    (d,) = torch.autograd.grad(rms_norm(row.expand(6, 50), w, eps=EPS).sum(), row)
    (e,) = torch.autograd.grad(rms_norm(row, w, eps=EPS).sum(), row)
    assert torch.all((d - 6 * e).abs() <= 6 * 200 * tol.U)


def test_special_rows():
    """NaN and infinity stay in their rows, zeros give zeros."""
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce("rms_norm special rows")
    for d in (40, 3000, 40000):
        x = torch.randn(5, d)
        x[0], x[1, 3], x[2, 5] = 0.0, float("nan"), float("inf")
        x = x.cuda()
        w = torch.ones(d, device="cuda")
        y = rms_norm(x, w)
        assert torch.all(y[0] == 0) and torch.isnan(y[1]).all() and torch.isnan(y[2, 5])
        assert torch.all(y[2, :5] == 0) and torch.isfinite(y[3:]).all()
        codes, scales = rms_norm_quantized(x, w)
        assert torch.all(codes[0].float() == 0) and torch.isnan(codes[1].float()).all()
        assert torch.isfinite(codes[3:].float()).all()


def test_empty():
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce("rms_norm of no rows")
    x = torch.empty(0, 300, device="cuda", requires_grad=True)
    w = torch.ones(300, device="cuda", requires_grad=True)
    y, h = rms_norm(x, w, x)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == (0, 300) and torch.all(w.grad == 0)
    with torch.no_grad():
        codes, scales = rms_norm_quantized(x, w)
    assert codes.shape == (0, 300) and scales.shape == (0, 3)


def test_another_stream_and_repeats():
    announce("rms_norm on a side stream, twice")
    args = _inputs(700, 1300, (torch.bfloat16, torch.bfloat16, torch.bfloat16))
    first = _run(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = _run(*args)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_offsets_past_32_bits():
    from cases.rms_norm.op import rms_norm
    announce("rms_norm rows 2^31 numbers apart")
    far, d = 2 ** 31 + 24, 300
    buf = torch.empty(far + d, dtype=torch.bfloat16, device="cuda")
    x, _, w, _, _ = _inputs(2, d, (torch.bfloat16, None, torch.float32))
    buf[:d], buf[far:] = x[0].cuda(), x[1].cuda()
    y = rms_norm(buf.as_strided((2, d), (far, 1)), w.cuda(), eps=EPS)
    _check_forward(x, None, w, y, None)


def test_many_rows():
    """More rows than a launch has workgroups of 1024 threads: a head's numbers each."""
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    rows, d, few = (1 << 22) + 4099, 64, 3
    announce(f"rms_norm {rows} x {d}")
    x, _, w, dy, _ = _inputs(few, d, (torch.bfloat16, None, torch.float32))
    big = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    big[-few:] = x.cuda()
    big.requires_grad_(True)
    wd = w.cuda().requires_grad_(True)
    dyd = torch.zeros_like(big)
    dyd[-few:] = dy.cuda()
    y = rms_norm(big, wd, eps=EPS)
    dx, dw = torch.autograd.grad(y, (big, wd), dyd)
    assert torch.all(y[:-few] == 0) and torch.all(dx[:-few] == 0)
    _, wh, r = _check_forward(x, None, w, y[-few:].detach(), None)
    _check_backward(x, None, w, dy, None, wh, r, dx[-few:], None, dw)
    with torch.no_grad():
        codes, scales = rms_norm_quantized(big, wd, eps=EPS)
        last = rms_norm_quantized(big[-few:], wd, eps=EPS)
    assert torch.equal(codes[-few:].view(torch.uint8), last[0].view(torch.uint8))
    assert torch.equal(scales[-few:].view(torch.uint8), last[1].view(torch.uint8))
    assert torch.all(codes[:-few].view(torch.uint8) == 0)


def test_refusals():
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce("rms_norm refusals")
    x, w = torch.zeros(3, 5, device="cuda"), torch.ones(5, device="cuda")
    for bad in (lambda: rms_norm(x.cpu(), w), lambda: rms_norm(x, w.cpu()),
                lambda: rms_norm(x.double(), w), lambda: rms_norm(x, w[:4]),
                lambda: rms_norm(x, w, x[:2]), lambda: rms_norm(x, w, x.bfloat16()),
                lambda: rms_norm(x[:, :0], w[:0]), lambda: rms_norm(x, w, eps=0.0),
                lambda: rms_norm(x, w, eps=-1.0), lambda: rms_norm(x, w, eps=float("nan")),
                lambda: rms_norm(x, w.view(1, 5)), lambda: rms_norm(x, w, x.cpu()),
                lambda: rms_norm_quantized(x, w, scale_dtype=torch.bfloat16),
                lambda: rms_norm_quantized(x.clone().requires_grad_(True), w)):
        with pytest.raises(RuntimeError):
            bad()
