"""hip backend of MXFP4 quantisation: tb_mxfp4_quant in libtbhip.so.

run(x) returns (codes uint8 [.., K / 2], scales uint8 [.., K / 32]) of x [.., K]
(float32, float16 or bfloat16, K a multiple of 32): per 32 channels the scale
2^(floor(log2(largest magnitude)) - 2), held to 2^-127 .. 2^127, codes rounded to
nearest even, beyond 6 to 6 (tilebench_amd.experts says how both are stored).
A block with inf or NaN reads back as NaN.

gated=True takes x [.., 2 K], gate then up, and quantises silu(gate) * up, the
step between an expert layer's products; codes and scales are those of the
product in 64 bits.
"""
import torch

from tilebench_amd import experts, paged
from tilebench_amd import runtime as rt

rt.load_library()

_last_config = None


def check(x, gated=False):
    """K of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "mxfp4_quant"
    if x.dtype not in experts.DTYPES:
        raise TypeError(f"{op}: x must be float32, float16 or bfloat16")
    if x.dim() < 2:
        raise ValueError(f"{op}: x must have two or more dimensions")
    K, rest = divmod(x.shape[-1], 2) if gated else (x.shape[-1], 0)
    if rest or K < experts.BLOCK or K % experts.BLOCK:
        raise ValueError(f"{op}: need a multiple of {experts.BLOCK} channels a row (got {x.shape[-1]}"
                         f"{', gate and up' if gated else ''})")
    return K


def run(x: torch.Tensor, gated: bool = False, **kwargs):
    global _last_config
    rt.require_device(x)
    K = check(x, gated)
    lead = x.shape[:-1]
    codes = x.new_empty((*lead, K // 2), dtype=torch.uint8)
    scales = experts.empty_scales(lead, K, x.device)
    if codes.numel():
        x = paged.aligned_rows(x if x.dim() == 2 else x.flatten(0, -2), 16 // x.element_size())
        rt.call("tb_mxfp4_quant", x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.shape[0], K, x.stride(0),
                -(-K // 512) * 16, gated, experts.DTYPES[x.dtype], rt.stream_handle(x.get_device()))
    _last_config = {"kernel": "mxfp4_quant_kernel", "lanes_per_block": 4, "block": 256}
    return codes, scales


def get_last_config():
    return _last_config
