"""Token log-probabilities on the GPU against the float64 oracle: widths around
every kernel's edges, the three types, layouts of the rows, and rows of
infinities, lowest values and NaN.  Bounds: operator_tolerances.py."""

import pytest
import torch

import operator_tolerances as tol
from conftest import announce
from oracle import token_rows as orow

pytestmark = pytest.mark.gpu

# windows hold 4 or 8 elements; the kernels change at 256, 512, 1024 and 16384 windows
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 63, 65, 255, 257, 1000, 1023, 1025, 2048, 2049, 4095, 4097, 8193,
          8200, 33001, 65537, 131073]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + v)
    x = (torch.randn(rows, v, generator=g) * 3).to(dtype)
    labels = torch.randint(0, v, (rows,), generator=g)
    labels[0] = v - 1
    if rows > 2:
        labels[1] = 0
        labels[2] = orow.IGNORE
    return g, x, labels


def _check(x, labels, up, logp, d, temperature=1.0):
    want = orow.logp(x, labels, temperature)
    keep = labels != orow.IGNORE
    err = (logp.cpu().double() - want).abs()
    assert torch.all(err <= torch.where(keep, tol.logp_error(x, labels, want, temperature), 0.0))
    if d is None:
        return
    wd = orow.dlogits(x, labels, up, temperature)
    err = (d.cpu().double() - wd).abs()
    bound = tol.dlogits_error(x, labels, up, torch.zeros(len(labels)), wd, d.dtype, temperature)
    assert torch.all(err <= torch.where(keep[:, None], bound, 0.0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("v", WIDTHS)
def test_widths(v, dtype):
    from cases.token_logp.op import token_logp
    announce(f"token_logp width {v} {dtype}")
    rows = 6 if v < 5000 else 3
    g, x, labels = _inputs(rows, v, dtype)
    up = torch.randn(rows, generator=g)
    xd = x.cuda().requires_grad_(True)
    logp = token_logp(xd, labels.cuda())
    assert logp.dtype == torch.float32 and logp.shape == (rows,)
    (d,) = torch.autograd.grad(logp, xd, up.cuda())
    assert d.dtype == dtype and d.is_contiguous()
    _check(x, labels, up, logp.detach(), d)
    with torch.no_grad():
        assert torch.equal(token_logp(xd, labels.cuda()), logp)


@pytest.mark.parametrize("rows", [1, 1023, 1025, 5000])
@pytest.mark.parametrize("v", [12, 700, 4100, 9001])
def test_many_rows(rows, v):
    """Rows on both sides of where a wave, a workgroup of 256 and one of 1024 take over."""
    from cases.token_logp.op import token_logp
    announce(f"token_logp {rows} rows of {v}")
    if rows * v > 1 << 24:
        rows = (1 << 24) // v
    g, x, labels = _inputs(rows, v, torch.bfloat16, seed=rows)
    up = torch.randn(rows, generator=g)
    xd = x.cuda().requires_grad_(True)
    logp = token_logp(xd, labels.cuda(), temperature=0.7)
    (d,) = torch.autograd.grad(logp, xd, up.cuda())
    _check(x, labels, up, logp.detach(), d, 0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", ["next_token", "rows_apart", "offset", "columns", "expanded",
                                    "four", "vector", "transposed"])
def test_layouts(layout, dtype):
    from cases.token_logp.op import token_logp
    announce(f"token_logp layout {layout} {dtype}")
    g = torch.Generator().manual_seed(3)
    v = 301
    if layout == "next_token":
        x = torch.randn(3, 6, v, generator=g).to(dtype).cuda()[:, :-1]
    elif layout == "rows_apart":
        x = torch.randn(5, 2 * v, generator=g).to(dtype).cuda()[:, 7:7 + v]
    elif layout == "offset":
        x = torch.randn(5 * v + 1, generator=g).to(dtype).cuda()[1:].view(5, v)
    elif layout == "columns":
        x = torch.randn(5, 2 * v, generator=g).to(dtype).cuda()[:, ::2]
    elif layout == "expanded":
        x = torch.randn(1, v, generator=g).to(dtype).cuda().expand(5, v)
    elif layout == "four":
        x = torch.randn(2, 3, 2, v, generator=g).to(dtype).cuda()
    elif layout == "vector":
        x = torch.randn(v, generator=g).to(dtype).cuda()
    else:
        x = torch.randn(4, 3, v, generator=g).to(dtype).cuda().transpose(0, 1)
    shape = x.shape[:-1]
    labels = torch.randint(0, v, shape, generator=g)
    up = torch.randn(shape, generator=g)
    leaf = x.detach().requires_grad_(True)
    logp = token_logp(leaf, labels.cuda(), temperature=1.3)
    assert logp.shape == shape
    (d,) = torch.autograd.grad(logp, leaf, up.cuda())
    assert d.shape == x.shape
    _check(x.cpu().reshape(-1, v), labels.reshape(-1), up.reshape(-1), logp.detach().reshape(-1),
           d.reshape(-1, v), 1.3)


def test_gradient_of_a_broadcast_row():
    """Gradients of one row used for all tokens add up."""
    from cases.token_logp.op import token_logp
    announce("token_logp broadcast gradient")
    g = torch.Generator().manual_seed(9)
    base = torch.randn(1, 64, generator=g).cuda().requires_grad_(True)
    labels = torch.randint(0, 64, (9,), generator=g)
    token_logp(base.expand(9, 64), labels.cuda()).sum().backward()
    want = orow.dlogits(base.detach().cpu().expand(9, 64), labels, torch.ones(9)).sum(0)
    assert torch.all((base.grad[0].cpu().double() - want).abs() <= 9 * 200 * tol.U)


def test_offsets_past_32_bits():
    from cases.token_logp.op import token_logp
    announce("token_logp rows 2^31 elements apart")
    v, far = 1000, 2 ** 31 + 11
    buf = torch.empty(far + v, dtype=torch.bfloat16, device="cuda")
    g, x, labels = _inputs(2, v, torch.bfloat16)
    buf[:v], buf[far:] = x[0].cuda(), x[1].cuda()
    view = buf.as_strided((2, v), (far, 1)).requires_grad_(True)
    logp = token_logp(view, labels.cuda())
    _check(x, labels, None, logp.detach(), None)


@pytest.mark.parametrize("v", [5, 300, 5000, 40000])
def test_infinities_and_lowest_values(v):
    from cases.token_logp.op import logp_backward, logp_forward
    announce(f"token_logp special rows of {v}")
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        _, x, labels = _inputs(9, v, dtype)
        labels[:] = torch.arange(9) % v
        labels[2] = orow.IGNORE
        x[0, 1:] = -float("inf")           # one class left, the label
        x[1, 2:] = low                     # masked by the lowest value
        x[2] = float("nan")                # ignored
        x[3] = -float("inf")               # nothing left: 0 / 0
        x[4] = low                         # all masked by the lowest value: uniform
        x[5, 0] = float("inf")
        x[6, 0] = float("nan")
        x[7, labels[7]] = -float("inf")    # the label masked
        labels[8] = v                      # no such class
        for temperature in (1.0, 0.5):
            xd, ld = x.cuda(), labels.cuda()
            logp, stats = logp_forward(xd, ld, temperature, keep_stats=True)
            d = logp_backward(xd, ld, stats, torch.ones(9, device="cuda"), temperature)
            logp, d = logp.cpu(), d.cpu().double()
            assert logp[0] == 0 and torch.all(d[0] == 0)
            assert logp[2] == 0 and torch.all(d[2] == 0)
            for r in (3, 5, 6, 8):
                assert torch.isnan(logp[r]) and torch.isnan(d[r]).any()
            assert abs(logp[4].item() + torch.log(torch.tensor(float(v))).item()) <= 40 * tol.U
            assert torch.all((d[4] + 1 / (v * temperature) -
                              (torch.arange(v) == labels[4]) / temperature).abs()
                             <= 2 * tol.TYPE_EPS[dtype] / temperature)
            assert logp[7] == -float("inf") and torch.isfinite(d[7]).all()
            two = x[1:2, :2].double() / temperature
            assert abs(logp[1] - (two[0, 1] - torch.logsumexp(two[0], 0))) <= 60 * tol.U * (
                1 + two.abs().max())
            assert torch.all(d[1, 2:] == 0)


def test_large_common_offset_costs_nothing():
    """Logits around 1e4 whose differences are exact: as around 0."""
    from cases.token_logp.op import token_logp
    announce("token_logp offset logits")
    g = torch.Generator().manual_seed(4)
    x = torch.randint(-64, 64, (4, 999), generator=g).float() / 16
    labels = torch.randint(0, 999, (4,), generator=g).cuda()
    a, b = token_logp(x.cuda(), labels), token_logp((x + 8192).cuda(), labels)
    assert torch.equal(a, b)


def test_empty():
    from cases.token_logp.op import token_logp
    announce("token_logp of no tokens")
    x = torch.empty(0, 50, device="cuda", requires_grad=True)
    logp = token_logp(x, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert logp.shape == (0,)
    logp.sum().backward()
    assert x.grad.shape == (0, 50)
    assert token_logp(torch.empty(3, 0, 8, device="cuda"),
                      torch.empty(3, 0, dtype=torch.int64, device="cuda")).shape == (3, 0)


def test_another_stream_and_repeats():
    from cases.token_logp.op import token_logp
    announce("token_logp on a side stream, twice")
    g, x, labels = _inputs(64, 3001, torch.bfloat16)
    xd, ld = x.cuda(), labels.cuda()
    first = token_logp(xd, ld)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = token_logp(xd, ld)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, second)


def test_refusals():
    from cases.token_logp.op import token_logp
    announce("token_logp refusals")
    x, l = torch.zeros(3, 5, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: token_logp(x.cpu(), l), lambda: token_logp(x, l.cpu()),
                lambda: token_logp(x.double(), l), lambda: token_logp(x, l.int()),
                lambda: token_logp(x, l[:2]), lambda: token_logp(x[:, :0], l),
                lambda: token_logp(x, l, temperature=0.0),
                lambda: token_logp(x, l, temperature=float("nan")),
                lambda: token_logp(x, l, temperature=-1.0)):
        with pytest.raises(RuntimeError):
            bad()
