"""PyTorch reference of MXFP4 quantisation.

Per 32 channels e = floor(log2(absmax)) - 2 held to -127 .. 127, the scale byte
e + 127; codes of x * 2^-e to nearest even.  Gated values silu(gate) * up are
formed in 64 bits and not rounded in between.  Blocks with inf or NaN: scale 255,
codes 0.
"""
import torch

BLOCK = 32


def gate(x):
    g, u = x.double().chunk(2, dim=-1)
    return g / (1.0 + torch.exp(-g)) * u


def power(e):
    """2^e in 64 bits, from its bits (|e| <= 1022)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def run(x, gated=False, **kwargs):
    v = gate(x) if gated else x.double()
    v = v.unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(dim=-1)
    bad = ~torch.isfinite(v).all(dim=-1)
    e = torch.frexp(torch.where(bad, torch.ones_like(top), top))[1] - 3
    e = torch.where(top == 0, torch.full_like(e, -127), e).clamp(-127, 127)
    v = torch.where(bad[..., None], torch.zeros_like(v), v) * power(-e)[..., None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v) & ~bad[..., None]).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
