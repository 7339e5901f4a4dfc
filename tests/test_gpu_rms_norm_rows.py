"""Root-mean-square norm on the GPU: backwards whose workgroups take several rows,
gradients against differences, and what lies behind a row's codes.  Bounds:
layer_tolerances.py and layer_differences.py."""

import pytest
import torch

import layer_differences as ld
from conftest import announce
from test_gpu_rms_norm import _check_backward, _check_forward, _gpu, _inputs, _run

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
