"""PyTorch reference of rotary positions with several axes.

angle[t, i] = positions[axes[i], t] * inv_freq[i] in fp64 (an fp32 product loses
4e-3 rad at position 65536); cos and sin rounded to fp32, the rotation in fp32,
one rounding to the inputs' type.
"""
import torch


def table(positions, inv_freq, axes, inverse=False):
    """cos and sin [T, 1, pairs]."""
    p = positions.double().reshape(-1, positions.shape[-1])
    axes = torch.zeros_like(inv_freq, dtype=torch.long) if axes is None else axes.long()
    angle = p[axes].t() * inv_freq.double()
    sin = torch.sin(angle).float()
    return torch.cos(angle).float()[:, None], (-sin if inverse else sin)[:, None]


def rotate(x, cos, sin, interleaved=False):
    """fp32 values of x [T, H, D] rotated."""
    x, R = x.float(), 2 * cos.shape[-1]
    head = x[..., :R]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, dim=-1)
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((head, x[..., R:]), dim=-1)


def run(q, k, positions, inv_freq, axes=None, interleaved=False, inverse=False, **kwargs):
    cos, sin = table(positions, inv_freq, axes, inverse)
    return tuple(None if x is None else rotate(x, cos, sin, interleaved).to(x.dtype) for x in (q, k))
