"""hip backend of reading MXFP4 back: tb_mxfp4_dequant in libtbhip.so.

run(codes uint8 [.., K / 2], scales uint8 [.., K / 32], dtype) returns values
[.., K] of dtype (float32, float16 or bfloat16): code times scale, rounded once
(tilebench_amd.experts says how both are stored).
"""
import torch

from tilebench_amd import experts
from tilebench_amd import runtime as rt

rt.load_library()

_last_config = None


def check(codes, scales, dtype=torch.bfloat16):
    """K of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "mxfp4_dequant"
    K = experts.check_matrix(op, "the matrix", codes, scales, None)
    if dtype not in experts.DTYPES:
        raise TypeError(f"{op}: the output must be float32, float16 or bfloat16")
    return K


def run(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16, **kwargs):
    global _last_config
    rt.require_device(codes, scales)
    K = check(codes, scales, dtype)
    out = codes.new_empty((*codes.shape[:-1], K), dtype=dtype)
    if out.numel():
        codes = experts.code_rows(codes)
        scales = scales if scales.dim() == 2 else scales.flatten(0, -2)
        M, S = scales.shape
        if (S > 1 and scales.stride(1) != 1) or (M > 1 and scales.stride(0) < S):
            scales = scales.contiguous()
        rt.call("tb_mxfp4_dequant", codes.data_ptr(), scales.data_ptr(), out.data_ptr(), M, K,
                scales.stride(0) if M > 1 else S, experts.DTYPES[dtype], rt.stream_handle(codes.get_device()))
    _last_config = {"kernel": "mxfp4_dequant_kernel", "block": 256}
    return out


def get_last_config():
    return _last_config
