"""Argument checks shared by the operators of the attention path (host side, no GPU).

A paged cache is one pool [pages, heads, page_size, head_dim] for the keys and
one for the values, in any memory order whose last dimension is contiguous
([pages, page_size, heads, head_dim] pools are passed as their permuted view,
pools that hold keys and values side by side as slices).  Slot s is row
s % page_size of page s // page_size.  A pool of float8_e4m3fn codes comes with
fp32 scales [pages, heads, page_size]: an element is its code times its row's
scale.
"""
from __future__ import annotations

import torch

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
MAX_HEAD_DIM = 512
MAX_AXES = 8
MAX_PAGE = 4096


def check_rotation(op, q, k, positions, inv_freq, axes):
    """(tokens, heads of q, heads of k, head_dim, rotated channels, axes) of a rotation."""
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError(f"{op}: q and k must be [tokens, heads, head_dim] with the same tokens and head_dim")
    if q.dtype not in DTYPES or q.dtype == torch.float8_e4m3fn or (k is not None and k.dtype != q.dtype):
        raise TypeError(f"{op}: q and k must share one of float32, float16 and bfloat16")
    T, Hq, D = q.shape
    if positions.dtype != torch.int32 or inv_freq.dtype != torch.float32:
        raise TypeError(f"{op}: positions must be int32 and inv_freq float32")
    A = positions.shape[0] if positions.dim() == 2 else 1
    if positions.dim() not in (1, 2) or positions.shape[-1] != T or not 1 <= A <= MAX_AXES:
        raise ValueError(f"{op}: positions must be [tokens] or [axes, tokens] with 1 to {MAX_AXES} axes")
    pairs = inv_freq.numel()
    if inv_freq.dim() != 1 or pairs < 1 or 2 * pairs > D or D % 2 or D > MAX_HEAD_DIM:
        raise ValueError(f"{op}: inv_freq must be one value per rotated pair, at most head_dim / 2 of them "
                         f"(head_dim even and at most {MAX_HEAD_DIM})")
    if axes is None:
        if A != 1:
            raise ValueError(f"{op}: {A} axes of positions need the axis of every pair")
    elif axes.dtype != torch.int32:
        raise TypeError(f"{op}: axes must be int32")
    elif tuple(axes.shape) != (pairs,):
        raise ValueError(f"{op}: axes must be one axis per pair of inv_freq")
    if Hq < 1 or (k is not None and k.shape[1] < 1):
        raise ValueError(f"{op}: need at least one head")
    return T, Hq, 0 if k is None else k.shape[1], D, 2 * pairs, A


def check_cache(op, dtype, heads, head_dim, k_cache, v_cache, k_scale, v_scale):
    """(pages, page_size) of a cache that holds `heads` heads of `head_dim` for inputs of `dtype`."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError(f"{op}: k_cache and v_cache must be [pages, heads, page_size, head_dim] of one shape and "
                         "memory order")
    pages, h, page, d = k_cache.shape
    if h != heads or d != head_dim:
        raise ValueError(f"{op}: the cache holds {h} heads of {d}, the inputs have {heads} of {head_dim}")
    if not 1 <= page <= MAX_PAGE or page & (page - 1):
        raise ValueError(f"{op}: the page size must be a power of two up to {MAX_PAGE} (got {page})")
    if pages < 1 or pages * page >= 1 << 31:
        raise ValueError(f"{op}: a cache holds 1 to 2^31 - 1 slots (got {pages} pages of {page})")
    if k_cache.stride(3) != 1 or 0 in k_cache.stride():
        raise ValueError(f"{op}: the cache's last dimension must be contiguous and no dimension expanded")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (dtype, torch.float8_e4m3fn):
        raise TypeError(f"{op}: the caches must be {dtype} like the inputs, or float8_e4m3fn")
    if k_cache.dtype == torch.float8_e4m3fn:
        if k_scale is None or v_scale is None:
            raise ValueError(f"{op}: float8_e4m3fn caches need k_scale and v_scale")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise TypeError(f"{op}: scales must be float32")
        if tuple(k_scale.shape) != (pages, h, page) or k_scale.shape != v_scale.shape \
                or k_scale.stride() != v_scale.stride() or 0 in k_scale.stride():
            raise ValueError(f"{op}: scales must be [pages, heads, page_size] of one memory order, no dimension "
                             "expanded")
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"{op}: scales belong to float8_e4m3fn caches")
    return pages, page


def rows(x):
    """x with its last dimension contiguous."""
    return x if x.stride(-1) == 1 else x.contiguous()
