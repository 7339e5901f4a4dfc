"""Block-scaled products on the GPU: tile scales for vectors and batches."""

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
