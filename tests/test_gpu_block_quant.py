"""Matrices in e4m3 on the GPU against the oracle, to the last bit: sizes around
blocks, types, layouts, both directions, and blocks of infinities, NaN, zeros and
the smallest and largest numbers."""

import pytest
import torch

from conftest import announce
from oracle import layers as ol

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SCALES = [torch.float32, torch.float8_e8m0fnu]


def _numbers(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + m * 7 + k)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)


def _same(codes, scales, x, tiles, scale_dtype):
    want, s = ol.quantize(x, tiles, scale_dtype != torch.float32)
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == scale_dtype
    assert codes.shape == x.shape and scales.shape == s.shape
    got = codes.cpu().float().double()
    assert torch.equal(scales.cpu().float().double().nan_to_num(-1.0, -2.0),
                       s.float().double().nan_to_num(-1.0, -2.0))
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (2, 129), (7, 127), (16, 8), (17, 1000),
                                 (127, 130), (128, 128), (129, 257), (300, 515)])
def test_sizes(m, k, dtype, scale_dtype):
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce(f"quantize {m} x {k} {dtype} {scale_dtype}")
    x = _numbers(m, k, dtype)
    d = x.cuda()
    _same(*quantize_rows(d, scale_dtype), x, False, scale_dtype)
    codes, scales, codes_t, scales_t = quantize_rows(d, scale_dtype, transposed=True)
    _same(codes, scales, x, False, scale_dtype)
    _same(codes_t, scales_t, x.t(), False, scale_dtype)
    tiles = quantize_tiles(d, scale_dtype)
    _same(*tiles, x, True, scale_dtype)
    codes, scales, codes_t, scales_t = quantize_tiles(d, scale_dtype, transposed=True)
    _same(codes, scales, x, True, scale_dtype)
    assert torch.equal(codes_t.view(torch.uint8), codes.view(torch.uint8).t())
    assert torch.equal(scales_t.view(torch.uint8), scales.t().view(torch.uint8)) \
        if scale_dtype != torch.float32 else torch.equal(scales_t, scales.t())
    for c, n in ((codes, k), (codes_t, m)):       # up to the next 16, zeros
        whole = c.as_strided((c.size(0), -(-n // 16) * 16), c.stride()).view(torch.uint8)
        assert torch.all(whole[:, n:] == 0)


def test_many_rows():
    """More blocks than the smaller workgroups take, and more than one of a row."""
    from cases.block_quant.op import quantize_rows
    for m, k in ((70000, 160), (9000, 2050)):
        announce(f"quantize {m} x {k}")
        x = _numbers(64, k, torch.bfloat16).repeat(-(-m // 64), 1)[:m]
        codes, scales = quantize_rows(x.cuda(), torch.float32)
        want = quantize_rows(x[:64].cuda(), torch.float32)
        for part in (slice(0, 64), slice(m // 64 * 64 - 64, m // 64 * 64)):
            assert torch.equal(codes[part].float(), want[0].float())
            assert torch.equal(scales[part], want[1])


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
def test_every_half_rounds_to_the_nearest_code(scale_dtype):
    """All float16 numbers up to 448, in blocks whose scale is 1: the instruction's rounding."""
    from cases.block_quant.op import quantize_rows
    announce("quantize every float16")
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    v = v[v.float().abs() <= 448]
    x = torch.full((-(-v.numel() // 127), 128), 448.0, dtype=torch.float16)
    flat = torch.zeros(x.size(0) * 127, dtype=torch.float16)
    flat[:v.numel()] = v
    x[:, :127] = flat.view(-1, 127)
    codes, scales = quantize_rows(x.cuda(), scale_dtype)
    assert torch.all(scales.float() == 1)
    want = torch.from_numpy(ol.to_e4m3(x.double().numpy()))
    assert torch.equal(codes.cpu().float().double(), want)


@pytest.mark.parametrize("layout", ["columns", "rows_apart", "offset", "expanded", "transposed",
                                    "three", "vector", "reversed_copy"])
def test_layouts(layout):
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce(f"quantize layout {layout}")
    base = _numbers(40, 900, torch.bfloat16).cuda()
    x = {"columns": base[:, ::2], "rows_apart": base[::3, 5:305], "offset": base.view(-1)[1:3001].view(10, 300),
         "expanded": base[:1].expand(20, 900), "transposed": base.t(),
         "three": base.view(4, 10, 900), "vector": base[3],
         "reversed_copy": base.flip(0)}[layout]
    codes, scales = quantize_rows(x)
    assert scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
    _same(codes.reshape(-1, x.size(-1)), scales.reshape(-1, scales.size(-1)),
          x.cpu().reshape(-1, x.size(-1)), False, torch.float8_e8m0fnu)
    if x.dim() == 2:
        _same(*quantize_tiles(x), x.cpu(), True, torch.float8_e8m0fnu)


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
def test_special_blocks(scale_dtype):
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce(f"quantize special blocks {scale_dtype}")
    for dtype in TYPES:
        big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        x = _numbers(10, 400, dtype)
        x[0] = 0.0
        x[1, 3] = float("nan")
        x[2, 130] = float("inf")
        x[3, 200] = -float("inf")
        x[4, :128] = big
        x[5] = small
        x[6] = -small / 4
        x[7, 5] = big
        x[8] = float("nan")
        x[9, ::2] = -0.0
        _same(*quantize_rows(x.cuda(), scale_dtype), x, False, scale_dtype)
        for rows in (slice(0, 2), slice(2, 4), slice(4, 8), slice(8, 9), slice(0, 10)):
            part = x[rows]
            _same(*quantize_tiles(part.cuda(), scale_dtype), part, True, scale_dtype)
        got = quantize_rows(x.cuda(), scale_dtype, transposed=True)
        _same(*got[2:], x.t(), False, scale_dtype)


def test_empty():
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce("quantize nothing")
    codes, scales = quantize_rows(torch.empty(0, 300, device="cuda"))
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    codes, scales = quantize_tiles(torch.empty(0, 300, device="cuda"))
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    codes, scales = quantize_rows(torch.empty(2, 0, 300, device="cuda"))
    assert codes.shape == (2, 0, 300) and scales.shape == (2, 0, 3)
    got = quantize_rows(torch.empty(0, 300, device="cuda"), transposed=True)
    assert got[2].shape == (300, 0) and got[3].shape == (300, 0)


def test_offsets_past_32_bits():
    from cases.block_quant.op import quantize_rows
    announce("quantize rows 2^31 numbers apart")
    far, k = 2 ** 31 + 24, 300
    buf = torch.empty(far + k, dtype=torch.bfloat16, device="cuda")
    x = _numbers(2, k, torch.bfloat16)
    buf[:k], buf[far:] = x[0].cuda(), x[1].cuda()
    _same(*quantize_rows(buf.as_strided((2, k), (far, 1))), x, False, torch.float8_e8m0fnu)


@pytest.mark.parametrize("what", ["rows", "tiles"])
def test_more_than_2_to_the_31_numbers(what):
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce(f"quantize {what} of 140032 x 16384")
    m, k = 1094 * 128, 16384
    quantize = quantize_rows if what == "rows" else quantize_tiles
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(128, k, device="cuda").bfloat16()
    x[-128:] = last
    u8 = torch.uint8
    codes, s, codes_t, s_t = (t.view(u8) for t in quantize(x, transposed=True))
    want, ws, want_t, ws_t = (t.view(u8) for t in quantize(last, transposed=True))
    assert torch.equal(codes[-128:], want) and torch.equal(codes_t[:, -128:], want_t)
    assert torch.equal(s[-len(ws):], ws) and torch.equal(s_t[:, -1:], ws_t)
    assert torch.all(codes[:-128] == 0) and torch.all(codes_t[:, :-128] == 0)
    del x, codes, codes_t
    torch.cuda.empty_cache()


def test_another_stream():
    from cases.block_quant.op import quantize_rows
    announce("quantize on a side stream")
    x = _numbers(300, 500, torch.bfloat16).cuda()
    first = quantize_rows(x, transposed=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = quantize_rows(x, transposed=True)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(first, second))


def test_refusals():
    from cases.block_quant.op import quantize_rows, quantize_tiles
    announce("quantize refusals")
    x = torch.zeros(3, 5, device="cuda")
    for bad in (lambda: quantize_rows(x.cpu()), lambda: quantize_rows(x.double()),
                lambda: quantize_rows(x, torch.bfloat16), lambda: quantize_rows(x[:, :0]),
                lambda: quantize_rows(x[0], transposed=True), lambda: quantize_tiles(x[0]),
                lambda: quantize_tiles(x.view(1, 3, 5)), lambda: quantize_tiles(x, None),
                lambda: quantize_rows(torch.zeros((), device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
