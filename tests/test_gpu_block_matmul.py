"""Block-scaled products on the GPU against the float64 oracle: sizes around tiles,
blocks and the kernels' edges, both kinds of scales, rows' and tiles', layouts, and
the layer with its gradients.  Bounds: layer_tolerances.py."""

import pytest
import torch

import layer_tolerances as tol
from conftest import announce
from oracle import layers as ol

pytestmark = pytest.mark.gpu

SCALES = [torch.float32, torch.float8_e8m0fnu]
OUT = [torch.float32, torch.bfloat16, torch.float16]


def _numbers(m, k, seed):
    g = torch.Generator().manual_seed(seed + m * 31 + k)
    return torch.randn(m, k, generator=g) * torch.exp(0.5 * torch.randn(m, 1, generator=g))


def _operands(m, n, k, tiles, scale_dtype, seed=0):
    """GPU codes and scales of a and b, and what they stand for on the CPU."""
    from cases.block_quant.op import quantize_rows, quantize_tiles
    got = []
    for side, rows, t in ((0, m, tiles[0]), (1, n, tiles[1])):
        q = (quantize_tiles if t else quantize_rows)(_numbers(rows, k, seed + side).cuda(),
                                                     scale_dtype)
        got.append((q, ol.values(q[0].cpu(), q[1].cpu())))
    return got


def _check(out, a, b, dtype):
    want, size = ol.matmul(a, b)
    assert out.dtype == dtype and out.shape == want.shape
    err = (out.cpu().double() - want).abs()
    assert torch.all(err <= tol.matmul_error(a, b, size, want, dtype))


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("tiles", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 128), (1, 300, 1000), (5, 33, 129),
                                   (16, 17, 31), (17, 200, 4096), (37, 130, 5000), (64, 64, 257),
                                   (65, 127, 640), (129, 300, 130), (128, 128, 2048),
                                   (200, 513, 385), (260, 150, 9000)])
def test_sizes(m, n, k, tiles, scale_dtype):
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul {m} x {n} x {k} tiles {tiles} {scale_dtype}")
    ((a, av), (b, bv)) = _operands(m, n, k, tiles, scale_dtype)
    dtype = OUT[(m + n) % 3]
    out = block_matmul(*a, *b, out_dtype=dtype)
    assert out.is_contiguous()
    _check(out, av, bv, dtype)
    assert torch.equal(out, block_matmul(*a, *b, out_dtype=dtype))


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("tiles", [(False, True), (False, False)])
def test_many_tiles(tiles, scale_dtype):
    """Sizes that take the larger tile, ragged at every end."""
    from cases.block_matmul.op import block_matmul
    m, n, k = 3500, 3810, 400
    announce(f"block_matmul {m} x {n} x {k} tiles {tiles} {scale_dtype}")
    ((a, av), (b, bv)) = _operands(m, n, k, tiles, scale_dtype)
    out = block_matmul(*a, *b, out_dtype=torch.float32)
    rows = torch.cat([torch.arange(0, 40), torch.arange(250, 262), torch.arange(m - 30, m)])
    cols = torch.cat([torch.arange(0, 40), torch.arange(250, 262), torch.arange(n - 30, n)])
    _check(out[rows.cuda()][:, cols.cuda()], av[rows], bv[cols], torch.float32)
    whole = av.cuda() @ bv.cuda().t().contiguous()
    size = av.cuda().abs() @ bv.cuda().abs().t().contiguous()
    assert torch.all((out.double() - whole).abs() <=
                     tol.matmul_error(av, bv, size, whole, torch.float32))
    half = block_matmul(*a, *b)
    _check(half[rows.cuda()][:, cols.cuda()], av[rows], bv[cols], torch.bfloat16)


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("tiles", [(False, True), (False, False)])
@pytest.mark.parametrize("m,n,k", [
    (16, 16390, 1030),        # a token or a few: two blocks at a time, and one
    (1, 700, 16500),
    (50, 500, 9000),
    (17, 16390, 1030),        # few rows, many numbers of b: stages, one part
    (1, 14000, 2500),
    (13, 5000, 10300),
    (9, 13000, 2700),
    (40, 4099, 4111),         # and parts of k
    (64, 1200, 14345),
    (300, 1100, 1111),        # small products, with parts of k and without
    (65, 130, 384),
    (230, 128, 6016),
    (66, 33, 64),
    (700, 2500, 200),         # tiles of 128, with fewer blocks than stages and more
    (520, 2100, 515),
    (900, 1500, 890),
    (1300, 3100, 515),        # of 256 x 128
    (2100, 3000, 900),
    (2100, 4000, 300),
    (4100, 4000, 130),        # of 256
    (3500, 4000, 600),
])
def test_every_kernel(m, n, k, tiles, scale_dtype):
    """Sizes that take each kernel, ragged at every end: all against 64 bits, 16-bit results also
    against the float32 ones."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul kernels {m} x {n} x {k} tiles {tiles} {scale_dtype}")
    ((a, av), (b, bv)) = _operands(m, n, k, tiles, scale_dtype)
    out = block_matmul(*a, *b, out_dtype=torch.float32).double()
    av, bv = av.cuda(), bv.cuda()
    want, size = av @ bv.t().contiguous(), av.abs() @ bv.abs().t().contiguous()
    assert torch.all((out - want).abs() <= tol.matmul_error(av, bv, size, want, torch.float32))
    # seven of eight products are off by 2^-13 of the largest, which their sum of magnitudes bounds
    for dtype in (torch.bfloat16, torch.float16):
        half = block_matmul(*a, *b, out_dtype=dtype).double()
        err = tol.rounded(size * (2 * tol.U * (128 + 5 * (k // 128 + 1) + 16) + 7 * 2.0 ** -13), want,
                          dtype)
        assert torch.all((half - want).abs() <= err)
        # as a whole nearer: of independent numbers a result's variance is at least that of the
        # largest products, and that of what is dropped, evenly spread, 7 / 3 * 2^-26 of it
        assert (half - want).norm() <= (tol.EPS[dtype] + 2.0 ** -12) * want.norm()


def test_exact_sums():
    """Small whole numbers: every sum is exact in 32 bits, and eight products in 13, so the answers
    are equal, to their last rounding."""
    from cases.block_matmul.op import block_matmul
    announce("block_matmul of whole numbers")
    g = torch.Generator().manual_seed(3)
    for m, n, k in ((3, 40, 700), (50, 100, 1200), (150, 300, 500), (1300, 2600, 300)):
        a, b = (torch.randint(-8, 9, (r, k), generator=g).float() for r in (m, n))
        one = [torch.ones(r, -(-k // 128)) for r in (m, n)]
        for dtype in SCALES:
            ca, cb = (t.cuda().to(torch.float8_e4m3fn) for t in (a, b))
            for kind in OUT:
                out = block_matmul(ca, one[0].to(dtype).cuda(), cb, one[1].to(dtype).cuda(),
                                   out_dtype=kind)
                assert torch.equal(out.cpu(), (a @ b.t()).to(kind))


def test_scales_of_every_block():
    """A one in each operand and scales that are all different: which scale goes where."""
    from cases.block_matmul.op import block_matmul
    announce("block_matmul scales")
    g = torch.Generator().manual_seed(4)
    for m, n in ((20, 300), (150, 300)):
        k = 5 * 128
        codes = [torch.zeros(r, k) for r in (m, n)]
        at = 128 * torch.randint(0, 5, (m,), generator=g) + torch.randint(0, 128, (m,), generator=g)
        codes[0][torch.arange(m), at] = 1.0
        codes[1][:] = 1.0
        for dtype in SCALES:
            for tiles in (False, True):
                sa = torch.exp2(torch.randint(-9, 9, (m, 5), generator=g).float())
                sb = torch.exp2(torch.randint(-9, 9, (-(-n // 128) if tiles else n, 5),
                                              generator=g).float())
                for kind in (torch.float32, torch.bfloat16):
                    out = block_matmul(codes[0].cuda().to(torch.float8_e4m3fn), sa.to(dtype).cuda(),
                                       codes[1].cuda().to(torch.float8_e4m3fn), sb.to(dtype).cuda(),
                                       out_dtype=kind).cpu().float()
                    kb = at // 128
                    each = sb.repeat_interleave(128, 0)[:n] if tiles else sb
                    assert torch.equal(out, sa[torch.arange(m), kb][:, None] * each[:, kb].t())


@pytest.mark.parametrize("layout", ["sliced", "dense", "column_slice", "offset", "transposed",
                                    "three", "vector", "scales_dense", "scales_expanded"])
def test_layouts(layout):
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul layout {layout}")
    m, n, k = 30, 70, 300
    ((a, av), (b, bv)) = _operands(m, n, k, (False, True), torch.float32)
    (ac, asc), (bc, bsc) = a, b
    u8 = torch.uint8
    if layout == "sliced":               # every other row
        out = block_matmul(ac[::2], asc[::2], bc, bsc)
        return _check(out, av[::2], bv, torch.bfloat16)
    if layout == "dense":                # rows of 300 bytes
        ac = ac.view(u8).contiguous().view(ac.dtype)
        assert ac.stride(0) == 300
    elif layout == "column_slice":       # what follows a row's 300 codes is not zeros but NaN
        wide = torch.full((m, 512), 127, dtype=u8, device="cuda")
        wide[:, 16:316] = ac.view(u8)
        ac = wide.view(ac.dtype)[:, 16:316]
        wide = torch.full((n, 304), 255, dtype=u8, device="cuda")
        wide[:, :300] = bc.view(u8)
        bc = wide.view(bc.dtype)[:, :300]
    elif layout == "offset":             # off 16 bytes, and at the end of its memory
        flat = torch.zeros(m * 304 + 4, dtype=u8, device="cuda")[4:]
        v = flat.view(m, 304)[:, :300]
        v.copy_(ac.view(u8))
        ac = v.view(ac.dtype)
        flat = torch.zeros(n * 304 - 4, dtype=u8, device="cuda")
        v = flat.as_strided((n, 300), (304, 1))
        v.copy_(bc.view(u8))
        bc = v.view(bc.dtype)
    elif layout == "transposed":
        ac = ac.view(u8).t().contiguous().t().view(ac.dtype)
    elif layout == "three":
        three = _numbers(m, k, 0).cuda().view(5, 6, k)
        from cases.block_quant.op import quantize_rows
        out = block_matmul(*quantize_rows(three, torch.float32), bc, bsc)
        assert out.shape == (5, 6, n)
        return _check(out.view(m, n), av, bv, torch.bfloat16)
    elif layout == "vector":
        out = block_matmul(ac[3], asc[3], bc, bsc)
        assert out.shape == (n,)
        return _check(out[None], av[3:4], bv, torch.bfloat16)
    elif layout == "scales_dense":
        asc = asc.contiguous()
        bsc = bsc.t().contiguous().t()
    else:
        asc = asc[:1].expand(m, -1)
        av = ol.values(ac.cpu(), asc.cpu())
    _check(block_matmul(ac, asc, bc, bsc), av, bv, torch.bfloat16)


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("m", [3, 150])
def test_special_numbers(m, scale_dtype):
    """A NaN makes its row of the result NaN; an infinite or NaN scale too; zeros give zeros; the
    smallest scales are applied."""
    from cases.block_matmul.op import block_matmul
    from cases.block_quant.op import quantize_rows
    announce(f"block_matmul special numbers {m} {scale_dtype}")
    x, w = _numbers(m, 300, 0), _numbers(200, 300, 1)
    x[0, 299], x[1, 5], x[2] = float("nan"), float("inf"), 0.0
    a, b = (quantize_rows(t.cuda(), scale_dtype) for t in (x, w))
    for kind in OUT:
        out = block_matmul(*a, *b, out_dtype=kind).cpu()
        assert torch.isnan(out[:2]).all() and torch.all(out[2] == 0)
    if m > 3:
        out = block_matmul(*a, *b, out_dtype=torch.float32)
        _check(out[3:], ol.values(*(t.cpu()[3:] for t in a)),
               ol.values(*(t.cpu() for t in b)), torch.float32)
    tiny = quantize_rows((x[3:4] if m > 3 else w[:1]).cuda() * 2.0 ** -100, scale_dtype)
    out = block_matmul(*tiny, *b, out_dtype=torch.float32)
    _check(out, ol.values(*(t.cpu() for t in tiny)), ol.values(*(t.cpu() for t in b)), torch.float32)


@pytest.mark.parametrize("m", [3, 40, 150])
def test_scales_that_no_quantiser_gives(m):
    """The ends of the exponents' range: 2^-127 and 2^127."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul e8m0 ends {m}")
    n, k = 70, 400
    ((a, _), (b, _)) = _operands(m, n, k, (False, False), torch.float8_e8m0fnu)
    u8 = torch.uint8
    asc, bsc = a[1].clone().view(u8), b[1].clone().view(u8)
    bsc.copy_(torch.tensor([127, 120], dtype=u8, device="cuda")[torch.arange(n) % 2, None])
    bsc += 100
    asc[0] = 0
    kinds = [(asc, bsc, 0)]
    asc2, bsc2 = asc.clone(), bsc - 200
    asc2[0] = 254
    kinds.append((asc2, bsc2, 0))
    for sa, sb, row in kinds:
        sa, sb = sa.view(torch.float8_e8m0fnu), sb.view(torch.float8_e8m0fnu)
        av, bv = ol.values(a[0].cpu(), sa.cpu()), ol.values(b[0].cpu(), sb.cpu())
        for dtype in (torch.float32, torch.bfloat16):
            out = block_matmul(a[0], sa, b[0], sb, out_dtype=dtype)
            _check(out[row:row + 1], av[row:row + 1], bv, dtype)


@pytest.mark.parametrize("m,n,scale_dtype", [(3, 300, torch.float32),
                                             (3, 300, torch.float8_e8m0fnu),
                                             (260, 300, torch.float32),
                                             (260, 300, torch.float8_e8m0fnu),
                                             (700, 2100, torch.float8_e8m0fnu)])
def test_rows_far_apart(m, n, scale_dtype):
    """Rows the longest pitch apart: offsets within a tile of almost 32 bits."""
    from cases.block_matmul.op import LONGEST, block_matmul
    announce(f"block_matmul rows far apart {m} x {n} {scale_dtype}")
    k, far = 200, 2 * LONGEST
    ((a, av), (b, bv)) = _operands(m, n, k, (False, True), scale_dtype)

    def apart(c):
        buf = torch.empty(len(c) * far, dtype=torch.uint8, device="cuda")
        view = buf.as_strided(c.shape, (far, 1))
        view.copy_(c.view(torch.uint8))
        return view.view(torch.float8_e4m3fn)
    ac, bc = apart(a[0]), apart(b[0])
    assert ac.stride(0) == bc.stride(0) == far
    _check(block_matmul(ac, a[1], bc, b[1]), av, bv, torch.bfloat16)
    del ac, bc
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [2, 66])
def test_longest_rows(m):
    from cases.block_matmul.op import LONGEST, block_matmul
    announce(f"block_matmul {m} x 5 x {LONGEST}")
    ((a, av), (b, bv)) = _operands(2, 5, LONGEST, (False, False), torch.float8_e8m0fnu)
    pick = torch.arange(m) % 2
    ac = a[0].view(torch.uint8)[pick.cuda()].view(torch.float8_e4m3fn)
    asc = a[1].view(torch.uint8)[pick.cuda()].view(torch.float8_e8m0fnu)
    out = block_matmul(ac, asc, *b, out_dtype=torch.float32)
    assert torch.equal(out, out[:2][pick.cuda()])
    _check(out[:2], av, bv, torch.float32)
    with pytest.raises(RuntimeError, match="too large"):
        block_matmul(torch.zeros(1, LONGEST + 1, device="cuda").to(torch.float8_e4m3fn),
                     torch.ones(1, LONGEST // 128 + 1, device="cuda"),
                     torch.zeros(1, LONGEST + 1, device="cuda").to(torch.float8_e4m3fn),
                     torch.ones(1, LONGEST // 128 + 1, device="cuda"))


@pytest.mark.parametrize("m,n", [(70000, 32800), (3, 5000000)])
def test_large_results(m, n):
    """More than 2^31 numbers; more rows of b than 2^16 times 64."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul {m} x {n}")
    ((a, av), (b, bv)) = _operands(300, 300, 16, (False, False), torch.float8_e8m0fnu)
    u8 = torch.uint8

    def spread(q, rows):
        """Zeros, then the last of q's rows."""
        few = min(rows, 300)
        codes = torch.zeros(rows, 16, dtype=u8, device="cuda")
        codes[-few:] = q[0].view(u8)[-few:]
        scales = torch.full((rows, 1), 127, dtype=u8, device="cuda")
        scales[-few:] = q[1].view(u8)[-few:]
        return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), few
    ac, asc, rows = spread(a, m)
    bc, bsc, cols = spread(b, n)
    out = block_matmul(ac, asc, bc, bsc)
    _check(out[-rows:, -cols:], av[-rows:], bv[-cols:], torch.bfloat16)
    assert torch.all(out[:-rows] == 0) and torch.all(out[:, :-cols] == 0)
    del out
    torch.cuda.empty_cache()


def test_empty():
    from cases.block_matmul.op import block_linear, block_matmul
    from cases.block_quant.op import quantize_rows
    announce("block_matmul of nothing")
    a = quantize_rows(torch.empty(0, 300, device="cuda"))
    b = quantize_rows(torch.ones(7, 300, device="cuda"))
    assert block_matmul(*a, *b).shape == (0, 7) and block_matmul(*b, *a).shape == (7, 0)
    x = torch.empty(0, 300, device="cuda", requires_grad=True)
    w = torch.ones(7, 300, device="cuda", requires_grad=True)
    block_linear(x, w).sum().backward()
    assert x.grad.shape == (0, 300) and torch.all(w.grad == 0)


# ------------------------------------------------------------------------- layer
def _layer_want(x, w, dy, power2):
    q = lambda t, tiles=False: ol.values(*ol.quantize(t, tiles, power2))  # noqa: E731
    wq = q(w, True)
    return ((q(x), wq), (q(dy), wq.t()), (q(dy.t()), q(x.t())))


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)],
                         ids=lambda t: "-".join(str(v)[6:] for v in t))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 200, 130), (50, 129, 300), (129, 140, 1000),
                                   (1000, 150, 70)])
def test_layer(m, n, k, types, scale_dtype):
    from cases.block_matmul.op import block_linear, quantize_weight
    announce(f"block_linear {m} x {n} x {k} {types} {scale_dtype}")
    x, w = _numbers(m, k, 0).to(types[0]), _numbers(n, k, 1).to(types[1])
    dy = _numbers(m, n, 2).to(types[0])
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = block_linear(xd, wd, scale_dtype=scale_dtype)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    want = _layer_want(x, w, dy, scale_dtype != torch.float32)
    _check(y.detach(), *want[0], types[0])
    _check(dx, *want[1], types[0])
    _check(dw, want[2][0], want[2][1], types[1])
    q = quantize_weight(w.cuda(), scale_dtype)
    z = block_linear(xd, wd, q, scale_dtype)
    assert torch.equal(z, y)
    assert all(torch.equal(a, b) for a, b in
               zip(torch.autograd.grad(z, (xd, wd), dy.cuda()), (dx, dw)))
    with torch.no_grad():
        assert torch.equal(block_linear(xd, wd, scale_dtype=scale_dtype), y)
    for one, got in ((xd, dx), (wd, dw)):       # the other is frozen
        leaf = one.detach().requires_grad_(True)
        args = (leaf, wd.detach()) if one is xd else (xd.detach(), leaf)
        (d,) = torch.autograd.grad(block_linear(*args, scale_dtype=scale_dtype), leaf, dy.cuda())
        assert torch.equal(d, got)


def test_layer_of_sequences():
    from cases.block_matmul.op import block_linear
    announce("block_linear of [2, 5, 300]")
    x, w = _numbers(10, 300, 0).cuda(), _numbers(40, 300, 1).cuda().requires_grad_(True)
    leaf = x.view(2, 5, 300).requires_grad_(True)
    y = block_linear(leaf, w)
    assert y.shape == (2, 5, 40)
    dx, dw = torch.autograd.grad(y.sum(), (leaf, w))
    flat = x.detach().requires_grad_(True)
    z = block_linear(flat, w)
    fx, fw = torch.autograd.grad(z.sum(), (flat, w))
    assert torch.equal(y.view(10, 40), z) and torch.equal(dx.view(10, 300), fx) and \
        torch.equal(dw, fw)
    head = block_linear(leaf[:, :-1], w)             # rows that are not one after the other
    assert torch.equal(head, y[:, :-1])


def test_differences_on_the_grid():
    """Where every number is a code times one scale, the layer is bilinear and exact: differences
    of whole steps are its gradients."""
    from cases.block_matmul.op import block_linear
    announce("block_linear differences")
    g = torch.Generator().manual_seed(7)

    def whole(*shape):
        x = torch.randint(-4, 5, shape, generator=g).float()
        x[:, ::64] = 7.0
        return x.cuda()
    X, W = whole(70, 130), whole(150, 130)
    G = torch.randint(-4, 5, (70, 150), generator=g).float().cuda()
    G[:, ::64], G[::64] = 7.0, 7.0
    X.requires_grad_(True), W.requires_grad_(True)
    dX, dW = torch.autograd.grad(block_linear(X, W), (X, W), G)
    with torch.no_grad():
        for i, j in ((1, 1), (66, 77), (2, 129)):
            for M, d in ((X, dX), (W, dW)):
                ys = []
                for step in (1, -1):
                    moved = M.clone()
                    moved[i, j] += step
                    ys.append(block_linear(moved, W) if M is X else block_linear(X, moved))
                assert ((ys[0] - ys[1]).double() * G).sum() / 2 == d[i, j]


def test_another_stream():
    from cases.block_matmul.op import block_linear
    announce("block_linear on a side stream")
    x, w = _numbers(300, 1500, 0).cuda(), _numbers(200, 1500, 1).cuda()
    first = block_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = block_linear(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, second)


def test_refusals():
    from cases.block_matmul.op import block_linear, block_matmul, quantize_weight
    from cases.block_quant.op import quantize_rows
    announce("block_matmul refusals")
    a, sa = quantize_rows(torch.ones(3, 200, device="cuda"), torch.float32)
    b, sb = quantize_rows(torch.ones(5, 200, device="cuda"), torch.float32)
    x, w = torch.ones(3, 200, device="cuda"), torch.ones(5, 200, device="cuda")
    for bad in (lambda: block_matmul(a.cpu(), sa, b, sb), lambda: block_matmul(a, sa, b, sb.cpu()),
                lambda: block_matmul(x, sa, b, sb), lambda: block_matmul(a, sa.double(), b, sb),
                lambda: block_matmul(a, sa, b, sb.to(torch.float8_e8m0fnu)),
                lambda: block_matmul(a, sa[:, :1], b, sb), lambda: block_matmul(a, sa[:2], b, sb),
                lambda: block_matmul(a, sa, b[:, :100], sb), lambda: block_matmul(a, sa, b[0], sb),
                lambda: block_matmul(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0]),
                lambda: block_matmul(a, sa, b, sb, out_dtype=torch.float64),
                lambda: block_linear(x, w.cpu()), lambda: block_linear(x.double(), w),
                lambda: block_linear(x, w[:, :7]), lambda: block_linear(x, w[0]),
                lambda: block_linear(x, w, scale_dtype=torch.bfloat16),
                lambda: block_linear(x, w, quantize_weight(w[:4])),
                lambda: block_linear(x, w, quantize_weight(w, torch.float32))):
        with pytest.raises(RuntimeError):
            bad()
