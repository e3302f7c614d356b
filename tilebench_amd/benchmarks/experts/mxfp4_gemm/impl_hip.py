"""hip backend of the MXFP4 product: tb_mxfp4_gemm in libtbhip.so.

run(a, sa, w, sw, dtype) returns Y [M, N] = a [M, K] w [N, K]^T in float16 or
bfloat16: fp32 accumulation, one rounding.  a uint8 [M, K / 2] with sa uint8
[M, K / 32], w [N, K / 2] with sw [N, K / 32] (tilebench_amd.experts says how
they are stored), K any multiple of 32.  Codes that are not dense, and scales
whose rows do not start on 4 bytes, are copied in the call.
"""
import torch

from tilebench_amd import experts
from tilebench_amd import runtime as rt

rt.load_library()

_last_call = None  # (M, N, K)


def check(a, sa, w, sw, dtype=torch.bfloat16):
    """(M, N, K) of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "mxfp4_gemm"
    K = experts.check_matrix(op, "a", a, sa, 2)
    if experts.check_matrix(op, "w", w, sw, 2) != K:
        raise ValueError(f"{op}: a has {K} channels, w {2 * w.shape[1]}")
    experts.check_output(op, dtype)
    return a.shape[0], w.shape[0], K


def run(a: torch.Tensor, sa: torch.Tensor, w: torch.Tensor, sw: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
        **kwargs):
    global _last_call
    rt.require_device(a, sa, w, sw)
    M, N, K = check(a, sa, w, sw, dtype)
    Y = a.new_empty((M, N), dtype=dtype)
    if not (M and N):
        return Y
    a, w = experts.code_rows(a), experts.code_rows(w)
    sa, sa_row, _ = experts.scale_rows(sa)
    sw, sw_row, _ = experts.scale_rows(sw)
    rt.call("tb_mxfp4_gemm", a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), Y.data_ptr(), M, N, K, sa_row,
            sw_row, experts.DTYPES[dtype], rt.stream_handle(a.get_device()))
    _last_call = M, N, K
    return Y


def get_last_config():
    return _last_call and {**rt.gemm_tile(rt.OP_MXFP4, *_last_call), "BK": 256}
