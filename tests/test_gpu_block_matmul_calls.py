"""Block-scaled products on the GPU: tile scales for vectors and batches, a row of
scales cut from a wide matrix, and layers of millions of tokens."""

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
