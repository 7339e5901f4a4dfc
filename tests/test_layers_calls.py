"""What the 8-bit layers' operators hand to the library, with a recorder in its place:
no GPU."""

import pytest
import torch

from test_layers_in_use import recorded  # noqa: F401  (a fixture)

E4M3 = torch.float8_e4m3fn


def _codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


@pytest.mark.parametrize("lead", [(), (1,), (2, 75), (3, 1, 50), (0, 4)])
@pytest.mark.parametrize("tiles", [False, True])
def test_scales_of_vectors_and_batches(lead, tiles, recorded):  # noqa: F811
    """Of rows, or of tiles of 128 of all the rows."""
    from cases.block_matmul.op import block_matmul
    m = torch.Size(lead).numel()
    scales = torch.ones(-(-m // 128), 3) if tiles else torch.ones(*lead, 3)
    out = block_matmul(_codes(*lead, 384), scales, _codes(7, 384), torch.ones(7, 3))
    assert out.shape == (*lead, 7)
    if m == 0:
        assert not recorded
        return
    (entry, args), = recorded
    assert args[2] == scales.data_ptr() and args[3:5] == (3, 1)
    assert args[5] == tiles or m == 1             # one row: either
    assert args[15:18] == (m, 7, 384)


@pytest.mark.parametrize("scales", [(2, 2), (3, 3), (150, 3), (2, 75, 2), (1, 2, 3)])
def test_scales_of_other_shapes_are_refused(scales, recorded):  # noqa: F811
    from cases.block_matmul.op import block_matmul
    with pytest.raises(RuntimeError, match="a_scales must be"):
        block_matmul(_codes(2, 75, 384), torch.ones(scales), _codes(7, 384), torch.ones(7, 3))
    assert not recorded


@pytest.mark.parametrize("m,k,shape,strides", [
    (1, 384, (1, 3), (1 << 23, 1)),               # a row of a wide matrix
    (100, 384, (1, 3), (1 << 40, 1)),             # a row of tiles of one
    (5, 100, (5, 1), (1, 1 << 61)),               # one block: its stride is never taken
    (300, 384, (3, 3), (1 << 23, 1)),             # too far apart: copied
])
def test_strides_of_scales_that_are_taken_are_in_range(m, k, shape, strides, recorded):  # noqa: F811
    """A dimension of one may come with any stride; no offset is made of it."""
    from cases.block_matmul.op import LONGEST, block_matmul
    real = tuple(s if n > 1 else 0 for n, s in zip(shape, strides))
    last = sum((n - 1) * s for n, s in zip(shape, real))
    scales = torch.ones(last + 1).as_strided(shape, real)
    scales = scales.as_strided(shape, strides)
    block_matmul(_codes(m, k), scales, _codes(7, k), torch.ones(7, -(-k // 128)))
    (entry, args), = recorded
    row, block = args[3:5]
    assert 0 <= row <= LONGEST and 0 <= block <= LONGEST
    assert args[2] == scales.data_ptr() or shape == (3, 3)
