"""MXFP4 checkpoint weights in the layout that the products take without a copy (no GPU needed)."""
import pytest
import torch

from tilebench_amd import experts
from tilebench_amd import formats as F
from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_torch as dequant_ref


def weights(*shape, seed=0):
    """Codes in blocks [.., K/32, 16] and scales [.., K/32], dense, as files hold them."""
    g = torch.Generator().manual_seed(seed)
    blocks = (*shape[:-1], shape[-1] // 32)
    return (torch.randint(0, 256, (*blocks, 16), generator=g, dtype=torch.uint8),
            torch.randint(100, 140, blocks, generator=g, dtype=torch.uint8))


def taken_as_they_lie(w):
    return experts.code_rows(w.codes) is w.codes and experts.scale_rows(w.scales)[0] is w.scales


@pytest.mark.parametrize("shape", [(5, 32), (1, 96), (40, 2912), (3, 7, 2912), (2, 1, 96), (4, 6, 256), (1, 5, 736)])
def test_weights_are_laid_out_once(shape):
    codes, scales = weights(*shape)
    want = dequant_ref.values(codes.flatten(-2), scales)
    w = F.mxfp4_checkpoint_to_tb(codes, scales)
    assert isinstance(w, F.Mxfp4Weights) and w.codes.shape == (*shape[:-1], shape[-1] // 2)
    assert taken_as_they_lie(w) and torch.equal(dequant_ref.values(w.codes, w.scales), want)
    again = F.mxfp4_checkpoint_to_tb(w.codes, w.scales)                # rows, and what lies so already
    assert again.codes is w.codes and again.scales is w.scales
    # rows at odd addresses, as slices of a larger file's buffer
    room = torch.empty(codes.numel() + 3, dtype=torch.uint8)[3:].view(codes.shape).copy_(codes)
    odd = torch.empty(scales.numel() + 1, dtype=torch.uint8)[1:].view(scales.shape).copy_(scales)
    w = F.mxfp4_checkpoint_to_tb(room, odd)
    assert taken_as_they_lie(w) and torch.equal(dequant_ref.values(w.codes, w.scales), want)


def test_an_odd_number_of_blocks_a_row_would_be_copied_in_every_call():
    codes, scales = weights(3, 7, 2912)
    assert experts.scale_rows(scales)[0] is not scales


def test_torch_types_of_the_bytes_are_taken():
    codes, scales = weights(6, 96)
    want = F.mxfp4_checkpoint_to_tb(codes, scales)
    for c, s in (("float4_e2m1fn_x2", "uint8"), ("uint8", "float8_e8m0fnu")):
        if hasattr(torch, c) and hasattr(torch, s):
            got = F.mxfp4_checkpoint_to_tb(codes.flatten(-2).view(getattr(torch, c)), scales.view(getattr(torch, s)))
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("codes,scales,error", [
    (torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.uint8), TypeError),
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2), TypeError),
    (torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), ValueError),
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8), ValueError),
    (torch.zeros(4, 2, 16, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8), ValueError),
    (torch.zeros(32, dtype=torch.uint8), torch.zeros(2, dtype=torch.uint8), ValueError),
    (torch.zeros(2, 2, 4, 32, dtype=torch.uint8), torch.zeros(2, 2, 4, 2, dtype=torch.uint8), ValueError)])
def test_other_shapes_are_refused(codes, scales, error):
    with pytest.raises(error):
        F.mxfp4_checkpoint_to_tb(codes, scales)
