"""Pins the float64 oracles of the 8-bit layers' operators: torch's own e4m3
numbers, closed forms, autograd, central differences, and planted mistakes that
the comparisons must catch."""

import math

import numpy as np
import pytest
import torch

from oracle import layers as ol


def _all_codes():
    """The 254 e4m3 numbers."""
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    return v[~v.isnan()].double().numpy()


def test_e4m3_rounds_to_the_nearest_number():
    codes = np.unique(_all_codes())
    assert np.array_equal(ol.to_e4m3(codes), codes) and codes.max() == 448
    mid = (codes[1:] + codes[:-1]) / 2
    for v in (mid, np.nextafter(mid, 1e9), np.nextafter(mid, -1e9)):
        got = ol.to_e4m3(v)
        near = codes[np.abs(v[:, None] - codes[None]).argmin(1)]
        tie = np.isin(v, mid)
        assert np.array_equal(got[~tie], near[~tie])
        bits = torch.from_numpy(got[tie]).to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.all(bits % 2 == 0)                  # ties to even
    v = np.random.default_rng(0).standard_normal(100000) * np.exp2(
        np.random.default_rng(1).uniform(-12, 7, 100000))
    v = v.astype(np.float32).astype(np.float64)
    want = torch.from_numpy(v).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ol.to_e4m3(v), want)
    assert np.isnan(ol.to_e4m3([464.0, 1e9, np.inf, np.nan])).all()
    assert np.array_equal(ol.to_e4m3([463.9, -460.0]), [448.0, -448.0])


@pytest.mark.parametrize("power2", [False, True])
def test_scales(power2):
    a = np.float32([0, 1e-45, 2.0 ** -120, 448, np.nextafter(np.float32(448), np.float32(1e9)), 1,
                    3.4e38, 1.75, np.inf])
    s = ol.scale_of(a, power2)
    if power2:
        assert s[:3].tolist() == [2.0 ** -126] * 3 and s[3] == 1 and s[4] == 2
        assert s[5] == 2.0 ** -8 and s[7] == 2.0 ** -8 and s[6] == 2.0 ** 120
        assert math.isnan(s[8])
        for x, y in zip(a[2:8].tolist(), s[2:8].tolist()):
            assert x <= 448 * y and (x > 448 * y / 2 or y == 2.0 ** -126)
    else:
        assert s[0] == s[1] == 2.0 ** -126 and s[3] == 1 and math.isinf(s[8])
        assert np.all(np.abs(s[3:8] * 448 / a[3:8].astype(np.float64) - 1) <= 2.0 ** -24)


@pytest.mark.parametrize("power2", [False, True])
@pytest.mark.parametrize("tiles", [False, True])
def test_quantized_numbers_are_near(tiles, power2):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(150, 300, generator=g) * torch.exp(2 * torch.randn(150, 1, generator=g))
    codes, s = ol.quantize(x, tiles, power2)
    back = ol.values(codes, s)
    each = ol.spread(s, 150, 300)
    # half a step of four bits, or of the smallest numbers' step
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, each * 2.0 ** -10) * (1 + 2.0 ** -20)
    assert torch.all((back - x.double()).abs() <= bound)
    # planted: a scale twice as large
    wrong = ol.values(codes, 2 * s)
    assert not torch.all((wrong - x.double()).abs() <= bound)


def test_special_numbers_of_a_block():
    x = torch.ones(3, 256)
    x[0, 3], x[1, 130], x[2] = float("nan"), float("inf"), 0.0
    for power2 in (False, True):
        codes, s = ol.quantize(x, False, power2)
        assert torch.isnan(codes[0, 3]) and torch.isnan(codes[0]).sum() == 1
        assert torch.isnan(ol.values(codes, s)[1, 128:]).all()
        assert torch.isfinite(ol.values(codes, s)[1, :128]).all()
        assert torch.all(codes[2] == 0) and torch.all(s[2] == 2.0 ** -126)


def test_norm_against_autograd_and_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 37, generator=g, dtype=torch.float64)
    w = 1 + 0.1 * torch.randn(37, generator=g, dtype=torch.float64)
    dy, dh = (torch.randn(5, 37, generator=g, dtype=torch.float64) for _ in range(2))
    xx, ww = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def value(h, w):
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w
        return (y * dy).sum() + (h * dh).sum()
    gx, gw = torch.autograd.grad(value(xx, ww), (xx, ww))
    y, h, r = ol.norm(x, w)
    dx, dw = ol.norm_backward(dy, h, w, r, dh)
    assert torch.allclose(dx, gx, atol=1e-13) and torch.allclose(dw, gw, atol=1e-13)
    step = 1e-6
    for i in range(0, 37, 5):
        e = torch.zeros_like(x)
        e[2, i] = step
        assert abs((value(x + e, w) - value(x - e, w)) / (2 * step) - dx[2, i]) < 1e-8
        e = torch.zeros_like(w)
        e[i] = step
        assert abs((value(x, w + e) - value(x, w - e)) / (2 * step) - dw[i]) < 1e-8
    # planted: the mean left out, the weight twice
    assert not torch.allclose(r * dy * w + dh, gx, atol=1e-6)
    assert not torch.allclose(ol.norm_backward(dy * w, h, w, r, dh)[0], gx, atol=1e-6)


def test_norm_of_the_rounded_sum():
    x = torch.full((1, 4), 1.0).bfloat16()
    res = torch.full((1, 4), 2.0 ** -9).bfloat16()
    _, h, r = ol.norm(x, torch.ones(4), res)
    assert torch.all(h == 1.0) and abs(r.item() - 1 / math.sqrt(1 + 1e-6)) < 1e-12


@pytest.mark.parametrize("name", ["rms_norm", "block_quant", "block_matmul"])
def test_references_pass_their_own_parity(name):
    import importlib
    from framework.verify import verify_all
    sizes = (13, 40, 200) if name == "block_matmul" else (13, 300)
    case = importlib.import_module(f"cases.{name}").make_case(*sizes)
    assert verify_all(case, case.reference_forward, device="cpu")[0]


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu], ids=str)
def test_references_agree_with_the_oracle(scale_dtype):
    from cases.block_matmul import reference as bm
    from cases.block_quant import reference as bq
    g = torch.Generator().manual_seed(3)
    x = torch.randn(140, 200, generator=g)
    power2 = scale_dtype != torch.float32
    want = ol.values(*ol.quantize(x, False, power2))
    assert torch.equal(bq.reference_forward({"X": x}, {"scale_dtype": scale_dtype}).double(),
                       want.float().double())
    assert torch.equal(bm.rounded(x, 1, scale_dtype).double(), want.float().double())
    tiles = ol.values(*ol.quantize(x, True, power2))
    assert torch.equal(bm.rounded(x, 128, scale_dtype).double(), tiles.float().double())


def test_differences_of_the_layer_on_the_grid():
    """Where every number is a code times one scale, the layer is bilinear: differences of whole
    steps are its gradients."""
    from cases.block_matmul.reference import reference_forward
    g = torch.Generator().manual_seed(4)

    def whole(*shape):
        x = torch.randint(-4, 5, shape, generator=g).double()
        x[:, ::64] = 7.0            # the largest of every block: the scale does not move
        return x
    X, W = whole(3, 130), whole(5, 130)
    G = torch.randint(-4, 5, (3, 5), generator=g).double()
    G[:, 0], G[0] = 7.0, 7.0
    X.requires_grad_(True), W.requires_grad_(True)
    params = {"scale_dtype": torch.float8_e8m0fnu}
    dX, dW = torch.autograd.grad(reference_forward({"X": X, "W": W}, params), (X, W), G)
    for i, j in ((0, 1), (2, 77), (1, 129)):
        for M, d in ((X, dX), (W, dW)):
            up, down = M.detach().clone(), M.detach().clone()
            up[i, j] += 1
            down[i, j] -= 1
            pair = [reference_forward({"X": m if M is X else X.detach(),
                                       "W": m if M is W else W.detach()}, params)
                    for m in (up, down)]
            assert ((pair[0] - pair[1]) * G).sum() / 2 == d[i, j]
