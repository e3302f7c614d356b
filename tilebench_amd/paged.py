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
    shape, dtype = q.shape, q.dtype
    kshape = shape if k is None else k.shape
    if len(shape) != 3 or len(kshape) != 3 or kshape[0] != shape[0] or kshape[2] != shape[2]:
        raise ValueError(f"{op}: q and k must be [tokens, heads, head_dim] with the same tokens and head_dim")
    if dtype not in DTYPES or dtype is torch.float8_e4m3fn or (k is not None and k.dtype is not dtype):
        raise TypeError(f"{op}: q and k must share one of float32, float16 and bfloat16")
    T, Hq, D = shape
    if positions.dtype is not torch.int32 or inv_freq.dtype is not torch.float32:
        raise TypeError(f"{op}: positions must be int32 and inv_freq float32")
    at, freqs = positions.shape, inv_freq.shape
    A = at[0] if len(at) == 2 else 1
    if len(at) not in (1, 2) or at[-1] != T or not 1 <= A <= MAX_AXES:
        raise ValueError(f"{op}: positions must be [tokens] or [axes, tokens] with 1 to {MAX_AXES} axes")
    pairs = freqs[0] if len(freqs) == 1 else 0
    if pairs < 1 or 2 * pairs > D or D % 2 or D > MAX_HEAD_DIM:
        raise ValueError(f"{op}: inv_freq must be one value per rotated pair, at most head_dim / 2 of them "
                         f"(head_dim even and at most {MAX_HEAD_DIM})")
    if axes is None:
        if A != 1:
            raise ValueError(f"{op}: {A} axes of positions need the axis of every pair")
    elif axes.dtype is not torch.int32:
        raise TypeError(f"{op}: axes must be int32")
    elif axes.shape != freqs:
        raise ValueError(f"{op}: axes must be one axis per pair of inv_freq")
    if Hq < 1 or kshape[1] < 1:
        raise ValueError(f"{op}: need at least one head")
    return T, Hq, 0 if k is None else kshape[1], D, 2 * pairs, A


def _strides(x):
    """Strides but for dimensions of size 1, where they do not matter."""
    return [s for s, n in zip(x.stride(), x.shape) if n > 1]


def check_cache(op, dtype, heads, head_dim, k_cache, v_cache, k_scale, v_scale):
    """(pages, page_size) of a cache that holds `heads` heads of `head_dim` for inputs of `dtype`."""
    shape, strides, kind = k_cache.shape, k_cache.stride(), k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape or (v_cache.stride() != strides
                                                     and _strides(v_cache) != _strides(k_cache)):
        raise ValueError(f"{op}: k_cache and v_cache must be [pages, heads, page_size, head_dim] of one shape and "
                         "memory order")
    pages, h, page, d = shape
    if h != heads or d != head_dim:
        raise ValueError(f"{op}: the cache holds {h} heads of {d}, the inputs have {heads} of {head_dim}")
    if not 1 <= page <= MAX_PAGE or page & (page - 1):
        raise ValueError(f"{op}: the page size must be a power of two up to {MAX_PAGE} (got {page})")
    if pages < 1 or pages * page >= 1 << 31:
        raise ValueError(f"{op}: a cache holds 1 to 2^31 - 1 slots (got {pages} pages of {page})")
    if strides[3] != 1 or (0 in strides and 0 in _strides(k_cache)):
        raise ValueError(f"{op}: the cache's last dimension must be contiguous and no dimension expanded")
    if v_cache.dtype is not kind or (kind is not dtype and kind is not torch.float8_e4m3fn):
        raise TypeError(f"{op}: the caches must be {dtype} like the inputs, or float8_e4m3fn")
    if kind is torch.float8_e4m3fn:
        if k_scale is None or v_scale is None:
            raise ValueError(f"{op}: float8_e4m3fn caches need k_scale and v_scale")
        if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise TypeError(f"{op}: scales must be float32")
        order = k_scale.stride()
        if k_scale.shape != shape[:3] or v_scale.shape != shape[:3] \
                or (v_scale.stride() != order and _strides(v_scale) != _strides(k_scale)) \
                or (0 in order and 0 in _strides(k_scale)):
            raise ValueError(f"{op}: scales must be [pages, heads, page_size] of one memory order, no dimension "
                             "expanded")
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"{op}: scales belong to float8_e4m3fn caches")
    return pages, page


def rows(x):
    """x with its last dimension contiguous."""
    return x if x.stride(-1) == 1 else x.contiguous()


def aligned_rows(x, step):
    """x with its last dimension contiguous, rows that start on 16 bytes and strides in multiples of `step` elements."""
    x = rows(x)
    if any(s % step for s in x.stride()[:-1]) or x.data_ptr() % 16:
        # dimensions of size 1 keep any stride in clone() and contiguous()
        x = x.new_empty(x.shape).copy_(x)
    return x


def dense(x):
    """An empty dense tensor of x's shape, type and device."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)
