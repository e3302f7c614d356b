"""MXFP4 matrices and the steps between an expert layer's operators (host side).

An MXFP4 matrix [.., K] is a pair of uint8 tensors: codes [.., K / 2], channel
2 j in the low and 2 j + 1 in the high four bits of byte j, each an e2m1 value
(bit 3 the sign; 0, 0.5, 1, 1.5, 2, 3, 4, 6), and scales [.., K / 32], the
powers of two 2^(scale - 127) of 32 channels each (255: NaN).  A value is its
code times its scale.  mxfp4_quant makes such pairs; it pads rows of scales to
16 bytes, so that scales whose K / 32 is no multiple of 4 are a view that the
products take without a copy.
"""
from __future__ import annotations

import torch

from tilebench_amd import runtime as rt

BLOCK = 32
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def check_matrix(op, what, codes, scales, dims):
    """K of an MXFP4 matrix of `dims` dimensions (None: two or more)."""
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise TypeError(f"{op}: {what} must be uint8 codes and scales")
    shape = codes.shape
    if len(shape) != dims if dims else len(shape) < 2:
        raise ValueError(f"{op}: {what} must have {dims or 'two or more'} dimensions (got {len(shape)})")
    K = 2 * shape[-1]
    if K < BLOCK or K % BLOCK:
        raise ValueError(f"{op}: {what} must hold a multiple of {BLOCK} channels a row (got {K})")
    if scales.shape != (*shape[:-1], K // BLOCK):
        raise ValueError(f"{op}: {what} needs one scale for {BLOCK} channels: {[*shape[:-1], K // BLOCK]}, got "
                         f"{list(scales.shape)}")
    return K


def check_output(op, dtype):
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"{op}: the output must be float16 or bfloat16")


def empty_scales(lead, K, device):
    """Unset scales [*lead, K / 32] whose rows start on 16 bytes."""
    S = K // BLOCK
    return torch.empty((*lead, -(-S // 16) * 16), dtype=torch.uint8, device=device)[..., :S]


def code_rows(codes):
    """codes dense and 16-byte aligned."""
    codes = codes.contiguous()
    return codes if codes.data_ptr() % 16 == 0 else codes.clone()


def scale_rows(scales):
    """(scales, bytes between rows, bytes between matrices) of [rows, S] or [matrices, rows, S], rows on 4 bytes; copied
    where they lie otherwise."""
    S = scales.shape[-1]
    n = scales.shape[-2]
    many = scales.shape[0] if scales.dim() == 3 else 1
    row = scales.stride(-2) if n > 1 else -(-S // 4) * 4
    matrix = scales.stride(0) if many > 1 else n * row
    if scales.data_ptr() % 4 or (S > 1 and scales.stride(-1) != 1) or row % 4 or row < S or matrix % 4 \
            or matrix < (n - 1) * row + S:
        scales = empty_scales(scales.shape[:-1], S * BLOCK, scales.device).copy_(scales)
        row = -(-S // 16) * 16
        matrix = n * row
    return scales, row, matrix


def align(ids, experts: int):
    """(pairs int32 [T * k], offsets int32 [experts + 1]) of a routing's ids int32 [T, k].

    pairs holds the numbers t * k + j of the (token, slot) pairs, sorted by
    expert and by themselves; expert e has pairs[offsets[e]:offsets[e + 1]].  Ids
    outside [0, experts) are routed nowhere: the entries of pairs from
    offsets[experts] on are then not set.  pairs are the rows that
    moe_mxfp4_grouped_gemm gathers (with topk = k) or scatters."""
    if ids.dtype is not torch.int32 or ids.dim() != 2:
        raise TypeError("align: ids must be int32 [tokens, k]")
    if not 0 < experts <= 4096:
        raise ValueError(f"align: need 1 to 4096 experts (got {experts})")
    rt.require_device(ids)
    ids = ids.contiguous()
    pairs = torch.empty((ids.numel(),), dtype=torch.int32, device=ids.device)
    if not ids.numel():
        return pairs, torch.zeros((experts + 1,), dtype=torch.int32, device=ids.device)
    offsets = torch.empty((experts + 1,), dtype=torch.int32, device=ids.device)
    rt.call("tb_moe_align", ids.data_ptr(), ids.numel(), experts, pairs.data_ptr(), offsets.data_ptr(),
            rt.stream_handle(ids.get_device()))
    return pairs, offsets


def combine(y, ids, experts: int):
    """out [T, H]: each token's rows of y [T * k, H] added in fp32 in slot order, rounded once; ids int32 [T, k] outside
    [0, experts) are left out."""
    if y.dtype is not torch.float16 and y.dtype is not torch.bfloat16 or ids.dtype is not torch.int32:
        raise TypeError("combine: y must be float16 or bfloat16 and ids int32")
    if y.dim() != 2 or ids.dim() != 2 or y.shape[0] != ids.numel():
        raise ValueError("combine: y must be [tokens * k, H] with ids [tokens, k]")
    rt.require_device(y, ids)
    y, ids = y.contiguous(), ids.contiguous()
    T, k = ids.shape
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    if out.numel():
        rt.call("tb_moe_combine" if y.dtype is torch.float16 else "tb_moe_combine_bf16", y.data_ptr(), ids.data_ptr(),
                out.data_ptr(), T, k, experts, y.shape[1], rt.stream_handle(y.get_device()))
    return out
