"""PyTorch reference of the MXFP4 product: both operands' values (exact in fp32), their product in fp32 (or the type
asked for), one rounding."""
import torch

from tilebench_amd.benchmarks.experts.mxfp4_dequant.impl_torch import values


def run(a, sa, w, sw, dtype=torch.bfloat16, compute=torch.float32, **kwargs):
    return (values(a, sa).to(compute) @ values(w, sw).to(compute).t()).to(dtype)
