"""Root-mean-square norm on the GPU: backwards whose workgroups take several rows,
gradients against differences, what lies behind a row's codes, and sizes past a
launch's.  Bounds: layer_tolerances.py and layer_differences.py."""

import pytest
import torch

import layer_differences as ld
import layer_tolerances as tol
from conftest import announce
from oracle import layers as ol
from test_gpu_rms_norm import EPS, _check_backward, _check_forward, _gpu, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,d", [(1, 300), (2, 5000), (3000, 72), (2100, 700), (1500, 1500),
                                    (600, 9000), (300, 17000)])
def test_rows_on_both_sides_of_the_workgroups(rows, d):
    """On both sides of where a workgroup of the backward takes more than one."""
    announce(f"rms_norm {rows} x {d}")
    kind = (torch.bfloat16, torch.bfloat16, torch.float32)
    x, res, w, dy, dh = _inputs(rows, d, kind)
    y, h, dx, dres, dw = _run(x, res, w, dy, dh)
    _, wh, r = _check_forward(x, res, w, y, h)
    _check_backward(x, res, w, dy, dh, wh, r, dx, dres, dw)


@pytest.mark.parametrize("d", [4, 7])
def test_every_gradient_against_differences(d):
    from cases.rms_norm.op import rms_norm
    announce(f"rms_norm differences, rows of {d}")
    x, res, w, dy, dh = ld.inputs(2, d, d)
    xd, rd, wd = (t.cuda().requires_grad_(True) for t in (x, res, w))
    y, h = rms_norm(xd, wd, rd, eps=ld.EPS)
    dx, dres, dw = torch.autograd.grad((y, h), (xd, rd, wd), (dy.cuda(), dh.cuda()))
    assert torch.equal(dx, dres)
    got = {"x": dx.cpu().double(), "weight": dw.cpu().double()}

    def value(x, w):
        with torch.no_grad():
            y, h = rms_norm(x.cuda(), w.cuda(), rd.detach(), eps=ld.EPS)
        return (y.cpu().double() * dy).sum() + (h.cpu().double() * dh).sum()
    for (which, at), (_, bound) in ld.bounds(x, res, w, dy, dh).items():
        up, down = (value(*ld.moved(x, w, which, at, by)) for by in (ld.STEP, -ld.STEP))
        assert abs((up - down) / (2 * ld.STEP) - got[which][at]) <= bound


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu], ids=str)
@pytest.mark.parametrize("d", [1, 8, 13, 40, 300, 700, 1500, 2056, 3001, 5000, 9001, 20003, 40003])
def test_codes_behind_a_row_are_zeros(d, scale_dtype):
    """Also behind a row whose numbers are all NaN."""
    from cases.rms_norm.op import rms_norm_quantized
    announce(f"rms_norm_quantized padding {d} {scale_dtype}")
    x, res, w, _, _ = _inputs(6, d, (torch.bfloat16, torch.bfloat16, torch.float32))
    x[1, d // 2], x[2, 0], x[4] = float("nan"), float("inf"), float("nan")
    xd, rd, wd = _gpu(x, res, w)
    p = -(-d // 16) * 16
    for r in (None, rd):
        codes, scales = rms_norm_quantized(xd, wd, r, scale_dtype=scale_dtype)[:2]
        whole = codes.as_strided((6, p), (p, 1)).view(torch.uint8)
        assert torch.all(whole[:, d:] == 0)
        assert torch.isnan(codes.float()[[1, 4]]).all()
        assert torch.isfinite(codes.float()[[0, 3, 5]]).all()
        # blocks without a number have the least scale
        assert torch.all(scales.float()[[1, 4]] == 2.0 ** -126)


# a launch has 4.19 million workgroups of 1024 threads, 16.7 million of 256
@pytest.mark.parametrize("rows,d", [((1 << 22) + 777, 4104), ((1 << 24) + 555, 1030)])
def test_more_rows_than_a_launch_has_workgroups(rows, d):
    """Rows one number apart, so that all differ in little memory; the two halves alone give the same
    bits."""
    from cases.rms_norm.op import rms_norm, rms_norm_quantized
    announce(f"rms_norm {rows} x {d}")
    g = torch.Generator().manual_seed(d)
    buf = torch.randn(rows + d, generator=g).bfloat16().cuda()
    w = (1 + 0.2 * torch.randn(d, generator=g)).cuda().requires_grad_(True)
    x = buf.as_strided((rows, d), (1, 1))
    y = rms_norm(x, w, eps=EPS)
    pick = torch.cat([torch.arange(0, 3), torch.arange(1 << 22, (1 << 22) + 5) - 3,
                      torch.arange(rows - 5, rows)])
    few = torch.stack([buf[i:i + d] for i in pick.tolist()]).cpu()
    _check_forward(few, None, w.detach().cpu(), y.detach()[pick.cuda()], None)
    with torch.no_grad():
        codes, scales = rms_norm_quantized(x, w, eps=EPS)
        for a, b in ((0, rows // 2), (rows // 2, rows)):
            assert torch.equal(rms_norm(x[a:b], w, eps=EPS), y[a:b])
            c, s = rms_norm_quantized(x[a:b], w, eps=EPS)
            assert torch.equal(c.view(torch.uint8), codes[a:b].view(torch.uint8))
            assert torch.equal(s.view(torch.uint8), scales[a:b].view(torch.uint8))
            del c, s
    del codes, scales
    with torch.no_grad():           # with a residual, in 32 bits
        res = buf.float().flip(0).as_strided((rows, d), (1, 1))
        last = slice(rows - 5000, rows)
        for call in (rms_norm, rms_norm_quantized):
            got, want = call(x, w, res, eps=EPS), call(x[last], w, res[last], eps=EPS)
            for a, b in zip(got, want):
                assert torch.equal(a[last].view(torch.uint8) if "float8" in str(a.dtype) else a[last],
                                   b.view(torch.uint8) if "float8" in str(b.dtype) else b)
            del got, want
    # ones for the last rows' gradients: the others' are zeros
    dy = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    dy[-5:] = 1
    (dw,) = torch.autograd.grad(y, w, dy.expand(rows, d))
    last = few[-5:]
    _, wh, r = ol.norm(last, w.detach().cpu(), None, EPS)
    ones = torch.ones(5, d)
    _, want = ol.norm_backward(ones, wh, w.detach().cpu(), r)
    # the same additions as of all the rows, of which all but five are zeros
    assert torch.all((dw.cpu().double() - want).abs() <= tol.dw_error(ones, wh, r, want, torch.float32))
    del y, dy
    torch.cuda.empty_cache()


def test_a_weight_gradient_of_more_columns_than_a_launch_has():
    """More than 2^28 numbers a row, 16 a workgroup."""
    from cases.rms_norm.op import rms_norm
    d = (1 << 28) + 37
    announce(f"rms_norm 1 x {d}")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, d, generator=g, device="cuda").bfloat16()
    dy = torch.randn(1, d, generator=g, device="cuda").bfloat16()
    w = torch.ones(d, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(rms_norm(x, w, eps=EPS), w, dy)
    r = 1 / torch.sqrt(x.double().square().mean() + EPS)
    want = (dy.double() * x.double() * r)[0]
    # one row: a product of three numbers, of which rstd's error is its sum's, (adds + 2) / 2
    err = want.abs() * tol.U * ((tol.adds(d) + 2) / 2 + 8)
    assert torch.all((dw.double() - want).abs() <= tol.rounded(err, want, torch.float32))
    del x, dy, w, dw, want, err
    torch.cuda.empty_cache()
