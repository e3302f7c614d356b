"""Layouts that the MXFP4 products are given (host side, no GPU)."""
import pytest
import torch

from tilebench_amd import experts


def strided(shape, strides):
    """A tensor of these strides over pages that are only touched where it lies."""
    room = torch.empty(sum((n - 1) * s for n, s in zip(shape, strides)) + 1, dtype=torch.uint8)
    return room.as_strided(shape, strides).copy_(torch.arange(torch.Size(shape).numel()).view(shape) % 251)


@pytest.mark.parametrize("shape,strides,copied", [
    ((4, 8), (1 << 22, 1), True), ((4, 8), ((1 << 22) - 4, 1), False), ((3, 4, 8), (1 << 24, 1 << 22, 1), True),
    # rows below 4 MiB apart that span 2 GiB: gaps are left out, dense rows are as short as they can be
    ((1030, 8), (1 << 21, 1), True), ((1020, 8), (1 << 21, 1), False)])
def test_rows_of_scales_far_apart_are_copied(shape, strides, copied):
    s = strided(shape, strides)
    got, row, matrix = experts.scale_rows(s)
    assert (got is not s) == copied and torch.equal(got, s)
    assert row < 1 << 22 and row % 4 == 0 and got.stride(-2) == row and shape[-2] * row < 1 << 31
    assert len(shape) == 2 or got.stride(0) == matrix
