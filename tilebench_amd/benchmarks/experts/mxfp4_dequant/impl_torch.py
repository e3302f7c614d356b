"""PyTorch reference of reading MXFP4 back: code times 2^(scale - 127), rounded once to the type (255: NaN)."""
import torch

from tilebench_amd.benchmarks.experts.mxfp4_quant.impl_torch import BLOCK, power

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values(codes, scales):
    """Values [.., K] in 64 bits."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]
    scale = torch.where(scales == 255, float("nan"), power(scales.long() - 127))
    return (v.unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


def run(codes, scales, dtype=torch.bfloat16, **kwargs):
    # a product of at most 3 bits: fp32 holds it, so one rounding follows
    return values(codes, scales).float().to(dtype)
