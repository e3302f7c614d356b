"""MXFP4 matrices and the steps between an expert layer's operators (host side).

An MXFP4 matrix [.., K] is a pair of uint8 tensors: codes [.., K / 2], channel
2 j in the low and 2 j + 1 in the high four bits of byte j, each an e2m1 value
(bit 3 the sign; 0, 0.5, 1, 1.5, 2, 3, 4, 6), and scales [.., K / 32], the
powers of two 2^(scale - 127) of 32 channels each (255: NaN).  A value is its
code times its scale.  mxfp4_quant makes such pairs; it pads rows of scales to
16 bytes, so that scales whose K / 32 is no multiple of 4 are a view that the
products take without a copy (moved to another device they become dense:
formats.mxfp4_checkpoint_to_tb lays weights out where they are used).
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
    shape, blocks = codes.shape, scales.shape
    n = len(shape)
    if n != dims if dims else n < 2:
        raise ValueError(f"{op}: {what} must have {dims or 'two or more'} dimensions (got {n})")
    half = shape[-1]
    if half % 16 or not half:
        raise ValueError(f"{op}: {what} must hold a multiple of {BLOCK} channels a row (got {2 * half})")
    if len(blocks) != n or 16 * blocks[-1] != half or blocks[0] != shape[0] or (n > 2 and blocks[1:-1] != shape[1:-1]):
        raise ValueError(f"{op}: {what} needs one scale for {BLOCK} channels: {[*shape[:-1], half // 16]}, got "
                         f"{list(blocks)}")
    return 2 * half


def check_output(op, dtype):
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"{op}: the output must be float16 or bfloat16")


def empty_scales(lead, K, device):
    """Unset scales [*lead, K / 32] whose rows start on 16 bytes."""
    S = K // BLOCK
    step = -(-S // 16) * 16
    strides = [1]
    for n in reversed(lead):
        strides.append(step)
        step *= n
    return torch.empty_strided((*lead, S), strides[::-1], dtype=torch.uint8, device=device)


def code_rows(codes):
    """codes dense and 16-byte aligned."""
    if not codes.is_contiguous():
        codes = codes.contiguous()
    return codes if codes.data_ptr() % 16 == 0 else codes.clone()


def scale_rows(scales):
    """(scales, bytes between rows, bytes between matrices) of [rows, S] or [matrices, rows, S], rows on 4 bytes; copied
    where they lie otherwise, or so far apart that the kernels' 32-bit offsets do not reach them (rows 4 MiB apart, or gaps
    between rows that add up to 2 GiB)."""
    *_, n, S = shape = scales.shape
    strides = scales.stride()
    row = strides[-2] if n > 1 else -(-S // 4) * 4
    matrix = strides[0] if len(shape) == 3 and shape[0] > 1 else n * row
    if (row | matrix | scales.data_ptr()) % 4 or (strides[-1] != 1 and S > 1) or row < S or matrix < (n - 1) * row + S \
            or row >= 1 << 22 or (n * row >= 1 << 31 and row >= S + 16):
        scales = empty_scales(shape[:-1], S * BLOCK, scales.device).copy_(scales)
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
    [0, experts) are left out.  A y that does not start on 16 bytes, or whose H is no multiple of 8, is copied in the
    call."""
    if y.dtype is not torch.float16 and y.dtype is not torch.bfloat16 or ids.dtype is not torch.int32:
        raise TypeError("combine: y must be float16 or bfloat16 and ids int32")
    if y.dim() != 2 or ids.dim() != 2 or y.shape[0] != ids.numel():
        raise ValueError("combine: y must be [tokens * k, H] with ids [tokens, k]")
    rt.require_device(y, ids)
    T, k = ids.shape
    H = y.shape[1]
    if H % 8:
        y = torch.nn.functional.pad(y, (0, -H % 8))
    else:
        y = y.contiguous()
        y = y if y.data_ptr() % 16 == 0 else y.clone()
    ids = ids.contiguous()
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    if out.numel():
        rt.call("tb_moe_combine" if y.dtype is torch.float16 else "tb_moe_combine_bf16", y.data_ptr(), ids.data_ptr(),
                out.data_ptr(), T, k, experts, y.shape[1], rt.stream_handle(y.get_device()))
    return out if out.shape[1] == H else out[:, :H].contiguous()
