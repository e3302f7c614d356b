"""hip backend of appending to a paged cache: tb_rope_kv_append in libtbhip.so.

run(q, k, v, positions, inv_freq, axes, slots, k_cache, v_cache) rotates q and k
(as rotary_axes does), writes k and v of token t into slot slots[t] of the paged
caches (tilebench_amd.paged says how these are laid out) and returns
(q', k_cache, v_cache), the caches being the ones given.  Slots outside the
cache (-1 for the padding of a captured batch) write nothing.  A slot named by
two tokens of one call holds an unspecified mix of both; the others are not
affected.

float8_e4m3fn caches take fp32 k_scale and v_scale and store each row of a head
as codes of x / s with s = absmax / 448, the codes and scales of 64-bit arithmetic (a zero row
stores s = 0 and zero codes, a row with inf or NaN reads back as NaN); run then
returns (q', k_cache, v_cache, k_scale, v_scale).
"""
import torch

from tilebench_amd import paged
from tilebench_amd import runtime as rt

rt.load_library()

_last_config = None


def check(q, k, v, positions, inv_freq, axes, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """The sizes of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "rope_kv_append"
    if k is None or v is None:
        raise ValueError(f"{op}: k and v are required")
    sizes = paged.check_rotation(op, q, k, positions, inv_freq, axes)
    if q.dtype is torch.float32:
        raise TypeError(f"{op}: q, k and v must be float16 or bfloat16")
    if v.shape != k.shape:
        raise ValueError(f"{op}: k and v must have one shape")
    if v.dtype is not k.dtype or slots.dtype is not torch.int32:
        raise TypeError(f"{op}: v must have k's type and slots be int32")
    if slots.shape != q.shape[:1]:
        raise ValueError(f"{op}: slots must be one slot per token")
    return sizes + paged.check_cache(op, q.dtype, sizes[2], sizes[3], k_cache, v_cache, k_scale, v_scale)


def run(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, axes,
        slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale=None, v_scale=None,
        interleaved: bool = False, **kwargs):
    global _last_config
    rt.require_device(q, k, v, positions, inv_freq, axes, slots, k_cache, v_cache, k_scale, v_scale)
    T, Hq, Hkv, D, R, A, pages, page = check(q, k, v, positions, inv_freq, axes, slots, k_cache, v_cache, k_scale,
                                             v_scale)
    q_out = paged.dense(q)
    q, k, v = paged.rows(q), paged.rows(k), paged.rows(v)
    positions, inv_freq, slots = positions.contiguous(), inv_freq.contiguous(), slots.contiguous()
    axes = None if axes is None else axes.contiguous()
    qs, ks, vs, cs = q.stride(), k.stride(), v.stride(), k_cache.stride()
    ss = (0, 0, 0) if k_scale is None else k_scale.stride()
    rt.call("tb_rope_kv_append", q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), positions.data_ptr(),
            inv_freq.data_ptr(), rt.ptr(axes), slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            rt.ptr(k_scale), rt.ptr(v_scale), T, Hq, Hkv, D, R, A, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], pages,
            page, cs[0], cs[1], cs[2], *ss, paged.DTYPES[q.dtype], paged.DTYPES[k_cache.dtype], interleaved,
            rt.stream_handle(q.get_device()))
    _last_config = {"kernel": "rotate_heads", "block": 256}
    return (q_out, k_cache, v_cache) if k_scale is None else (q_out, k_cache, v_cache, k_scale, v_scale)


def get_last_config():
    return _last_config
