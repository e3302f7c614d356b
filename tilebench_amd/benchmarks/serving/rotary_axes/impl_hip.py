"""hip backend of rotary positions with several axes: tb_rotary_axes in libtbhip.so.

run(q, k, positions, inv_freq, axes) rotates q [T, Hq, D] and k [T, Hk, D] (k may
be None) in one launch and returns dense (q', k').  positions is int32 [axes, T]
(or [T] for one axis), inv_freq fp32 one value per rotated pair, axes int32 the
axis each pair follows (None: the first).  Pairs are (i, i + R/2), or (2i, 2i+1)
with interleaved=True; channels from 2 * len(inv_freq) on pass through.
inverse=True rotates by the negated angles, which undoes a rotation and is its
gradient: dq, dk = run(dq', dk', ..., inverse=True).
"""
import torch

from tilebench_amd import paged
from tilebench_amd import runtime as rt

rt.load_library()

_last_config = None


def run(q: torch.Tensor, k, positions: torch.Tensor, inv_freq: torch.Tensor, axes=None, interleaved: bool = False,
        inverse: bool = False, **kwargs):
    global _last_config
    rt.require_device(q, k, positions, inv_freq, axes)
    T, Hq, Hk, D, R, A = paged.check_rotation("rotary_axes", q, k, positions, inv_freq, axes)
    q_out = paged.dense(q)
    k_out = None
    kst = ksh = 0
    q = paged.rows(q)
    if k is not None:
        k = paged.rows(k)
        k_out = paged.dense(k)
        kst, ksh, _ = k.stride()
    qst, qsh, _ = q.stride()
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    axes = None if axes is None else axes.contiguous()
    rt.call("tb_rotary_axes", q.data_ptr(), q_out.data_ptr(), rt.ptr(k), rt.ptr(k_out), positions.data_ptr(),
            inv_freq.data_ptr(), rt.ptr(axes), T, Hq, Hk, D, R, A, qst, qsh, kst, ksh,
            paged.DTYPES[q.dtype], interleaved, inverse, rt.stream_handle(q.get_device()))
    _last_config = {"kernel": "rotate_heads", "block": 256}
    return (q_out, k_out)


def get_last_config():
    return _last_config
