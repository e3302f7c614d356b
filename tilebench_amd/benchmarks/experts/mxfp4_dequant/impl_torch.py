"""PyTorch reference of reading MXFP4 back: code times 2^(scale - 127), rounded once to the type (255: NaN)."""
import torch

from tilebench_amd.benchmarks.experts.mxfp4_quant.impl_torch import BLOCK, power


def values(codes, scales):
    """Values [.., K] in 64 bits.  No table from the host, so that a call can be captured."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    m = (code & 7).double()
    v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))  # 0, 0.5, 1, 1.5, 2, 3, 4, 6
    v = torch.where(code > 7, -v, v)
    scale = torch.where(scales == 255, float("nan"), power(scales.long() - 127))
    return (v.unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


def run(codes, scales, dtype=torch.bfloat16, **kwargs):
    # a product of at most 3 bits: fp32 holds it, so one rounding follows
    return values(codes, scales).float().to(dtype)
