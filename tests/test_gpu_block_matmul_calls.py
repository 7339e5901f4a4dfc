"""Block-scaled products on the GPU: tile scales for vectors and batches, a row of
scales cut from a wide matrix, layers of millions of tokens, and what 16-bit results
lose beside their rounding."""

import pytest
import torch

from conftest import announce
from test_gpu_block_matmul import SCALES, _check, _operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("lead", [(), (1,), (2, 75), (3, 1, 50), (1, 1, 130)])
def test_tile_scales_of_vectors_and_batches(lead, scale_dtype):
    """Tiles of 128 rows, counted over all of a's leading dimensions."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul tiles of {lead} {scale_dtype}")
    m = torch.Size(lead).numel()
    ((a, av), (b, bv)) = _operands(m, 70, 300, (True, True), scale_dtype)
    codes = a[0].view(torch.uint8).reshape(*lead, 300).view(a[0].dtype)
    out = block_matmul(codes, a[1], *b)
    assert out.shape == (*lead, 70)
    _check(out.view(m, 70), av, bv, torch.bfloat16)
    assert torch.equal(out.view(m, 70), block_matmul(*a, *b))


def test_a_row_of_scales_of_a_wide_matrix():
    from cases.block_matmul.op import LONGEST, block_matmul
    announce("block_matmul scales of one row")
    ((a, av), (b, bv)) = _operands(1, 40, 300, (False, True), torch.float32)
    wide = [torch.zeros(2 * LONGEST + 3, device="cuda").as_strided((1, 3), (2 * LONGEST, 1))
            for _ in range(2)]
    for to, s in zip(wide, (a[1], b[1])):
        to.copy_(s)
    assert wide[0].stride(0) > LONGEST
    _check(block_matmul(a[0], wide[0], b[0], wide[1]), av, bv, torch.bfloat16)


@pytest.mark.parametrize("frozen", [True, False])
def test_a_layer_of_more_tokens_than_a_row_has_numbers(frozen):
    """4.19 million is where dweight's sums end; without it the tokens are rows like any others."""
    from cases.block_matmul.op import LONGEST, block_linear
    m, n, k = LONGEST + 77, 24, 40
    announce(f"block_linear {m} x {n} x {k}")
    g = torch.Generator().manual_seed(2)
    few = torch.randn(300, k, generator=g).bfloat16()
    x = few.cuda().repeat(-(-m // 300), 1)[:m]
    w = torch.randn(n, k, generator=g).cuda()
    dy = torch.randn(300, n, generator=g).bfloat16()
    if frozen:
        x.requires_grad_(True)
    y = block_linear(x, w)
    part = x[:300].detach().requires_grad_(frozen)
    z = block_linear(part, w)
    assert torch.equal(y.detach(), z.detach().repeat(-(-m // 300), 1)[:m])
    if frozen:
        (dx,) = torch.autograd.grad(y, x, dy.cuda().repeat(-(-m // 300), 1)[:m])
        (dp,) = torch.autograd.grad(z, part, dy.cuda())
        assert torch.equal(dx, dp.repeat(-(-m // 300), 1)[:m])
    with pytest.raises(RuntimeError, match="too large"):
        block_linear(x, w.requires_grad_(True))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("m,n,k", [(64, 8192, 4096), (256, 4096, 4096), (1024, 2048, 2048),
                                   (2048, 2048, 1024)])
def test_what_16_bit_results_lose_as_a_whole(m, n, k, scale_dtype):
    """Of random numbers 16-bit results are off by their rounding, and before it by what the 8-bit
    instruction drops: e, a root mean square of 1.5e-5 of the results', here held to 2^-15, twice that.

    e is seen through the rounding: it changes a result only where it carries it over a border between
    two numbers, with a chance of |e| / step, and then moves the square of its error by 2 step a, a evenly
    in [0, |e|]: by e^2 in the mean.  So the squares of the errors exceed those of the rounded 64-bit
    results by the sum of e^2, give or take sqrt(4/3 step / |e| / N) of it over N results: 5 % for bfloat16
    (step up to 2^-7) and 2 % for float16 with 2^19 of them.  Losing two bits more is four times the
    bound."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul losses {m} x {n} x {k} {scale_dtype}")
    ((a, av), (b, bv)) = _operands(m, n, k, (False, True), scale_dtype)
    want = av.cuda() @ bv.cuda().t().contiguous()
    assert want.abs().max() < 65504
    for dtype in (torch.float16, torch.bfloat16):
        out = block_matmul(*a, *b, out_dtype=dtype).double()
        lost = (out - want).square().sum() - (want.to(dtype).double() - want).square().sum()
        share = (lost / want.square().sum()).item()
        print(f"{dtype}: {abs(share) ** 0.5:.2e}")
        assert share <= 2.0 ** -30


@pytest.mark.parametrize("scale_dtype", SCALES, ids=str)
@pytest.mark.parametrize("m,n,k", [(3, 300, 1000), (12, 13000, 2700), (40, 4099, 1030), (200, 300, 1500),
                                   (1300, 3100, 300), (3500, 4000, 200)])
def test_what_outliers_take_from_their_eight(m, n, k, scale_dtype):
    """In one eight of eight a product is 2^17 times the others and more, every second time beside one
    that cancels it: only what shares its eight loses bits, and no more than the bound."""
    from cases.block_matmul.op import block_matmul
    announce(f"block_matmul outliers {m} x {n} x {k} {scale_dtype}")
    g = torch.Generator().manual_seed(m + k)

    def codes(rows, flip):
        x = (0.25 + torch.rand(rows, k, generator=g)) * torch.sign(torch.randn(rows, k, generator=g))
        at = torch.arange(3, k - 8, 64)                  # one eight of eight, at any of its places
        at = at + torch.randint(-3, 4, at.shape, generator=torch.Generator().manual_seed(k))
        x[:, at] = 448.0
        pairs = at[::2]                                  # and one that cancels it, in the same eight
        x[:, pairs // 8 * 8 + (pairs + 1) % 8] = 448.0 * flip
        return x.to(torch.float8_e4m3fn)
    a, b = codes(m, 1.0), codes(n, -1.0)
    one = [torch.ones(r, -(-k // 128)).to(scale_dtype).cuda() for r in (m, -(-n // 128))]
    av, bv = a.double(), b.double()
    pick = [torch.unique(torch.cat([torch.arange(0, min(r, 60)), torch.arange(max(r - 60, 0), r)]))
            for r in (m, n)]
    for dtype in (torch.float16, torch.bfloat16):
        # 448 * 448 a block would leave float16's range: a's scales take it back
        out = block_matmul(a.cuda(), (one[0].float() * 2.0 ** -8).to(scale_dtype), b.cuda(), one[1],
                           out_dtype=dtype)
        _check(out[pick[0].cuda()][:, pick[1].cuda()], av[pick[0]] * 2.0 ** -8, bv[pick[1]], dtype)
