"""PyTorch reference of appending to a paged cache with the rotation on the way.

The rotation of rotary_axes/impl_torch.py; k and v rounded once into copies of
the caches (the caches given are left as they are).  float8_e4m3fn caches: per
token and head s = fp32(absmax) / 448, codes of the fp32 quotient x / s, zeros
where s is 0.
"""
import torch

from tilebench_amd.benchmarks.serving.rotary_axes.impl_torch import rotate, table


def quantise(x):
    """e4m3 codes and fp32 scales of the rows of fp32 x."""
    s = x.abs().amax(dim=-1) / 448.0
    q = torch.where(s[..., None] == 0, torch.zeros_like(x), x / s[..., None])
    return q.to(torch.float8_e4m3fn), s


def run(q, k, v, positions, inv_freq, axes, slots, k_cache, v_cache, k_scale=None, v_scale=None, interleaved=False,
        **kwargs):
    cos, sin = table(positions, inv_freq, axes)
    pages, _, page, _ = k_cache.shape
    keep = (slots >= 0) & (slots < pages * page)
    slots = slots[keep].long()
    at = slots // page, slots % page
    caches, scales = [], []
    for x, cache, scale in ((rotate(k, cos, sin, interleaved), k_cache, k_scale), (v.float(), v_cache, v_scale)):
        cache, x = cache.clone(), x[keep]
        if scale is not None:
            codes, s = quantise(x)
            cache.view(torch.uint8)[at[0], :, at[1]] = codes.view(torch.uint8)
            scales.append(scale.clone())
            scales[-1][at[0], :, at[1]] = s
        else:
            cache[at[0], :, at[1]] = x.to(cache.dtype)
        caches.append(cache)
    return (rotate(q, cos, sin, interleaved).to(q.dtype), *caches, *scales)
