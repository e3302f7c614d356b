"""hip backend of the experts' MXFP4 products: tb_moe_mxfp4_grouped_gemm in libtbhip.so.

run(a, sa, w, sw, offsets) returns Y [R, N]: rows offsets[e] .. offsets[e + 1] - 1
(int32 [E + 1], ascending from 0) are a's rows times w[e]^T, in dtype (float16
or bfloat16).  a uint8 [rows, K / 2] with sa [rows, K / 32], w [E, N, K / 2]
with sw [E, N, K / 32] (tilebench_amd.experts says how they are stored).

gather  int32 [R]: product row m takes row gather[m] // topk of a (negative or
        past its end: a row of zeros), so that tokens are quantised once and
        pairs' rows are gathered on the way.  None: row m, R = rows.
scatter int32 [R]: product row m goes to row scatter[m] of Y (outside it:
        nowhere; a row named twice holds values of either), times
        weights[that row] (float32 [R]) if given, before the rounding.
out     the Y [R, N] to write.  Rows that no product row goes to are left as
        they were, those of a Y made here not set.

tilebench_amd.experts.align makes offsets and the pairs to gather or scatter.
Offsets stay on the device and are held to 0 .. R there.
"""
import torch

from tilebench_amd import experts
from tilebench_amd import runtime as rt

rt.load_library()

_last_call = None  # (R, N, K, E)


def check(a, sa, w, sw, offsets, gather=None, topk=1, scatter=None, weights=None, dtype=torch.bfloat16, out=None):
    """(R, N, K, E) of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "moe_mxfp4_grouped_gemm"
    K = experts.check_matrix(op, "a", a, sa, 2)
    if experts.check_matrix(op, "w", w, sw, 3) != K:
        raise ValueError(f"{op}: a has {K} channels, w {2 * w.shape[2]}")
    experts.check_output(op, dtype)
    E, N = w.shape[:2]
    if offsets.dtype is not torch.int32 or (gather is not None and gather.dtype is not torch.int32) \
            or (scatter is not None and scatter.dtype is not torch.int32):
        raise TypeError(f"{op}: offsets, gather and scatter must be int32")
    if not 1 <= E <= 4096 or offsets.shape != (E + 1,):
        raise ValueError(f"{op}: need 1 to 4096 experts and offsets [experts + 1] (got {E} and {list(offsets.shape)})")
    if gather is not None and gather.dim() != 1:
        raise ValueError(f"{op}: gather must be one row of a (times topk) for every product row")
    R = a.shape[0] if gather is None else gather.shape[0]
    if type(topk) is not int or not 1 <= topk < 1 << 31:
        raise ValueError(f"{op}: topk must be a positive number")
    if gather is not None and a.shape[0] == 0 and R:
        raise ValueError(f"{op}: no rows to gather from")
    if scatter is not None and scatter.shape != (R,):
        raise ValueError(f"{op}: scatter must be one row of Y for each of the {R} product rows")
    if weights is not None:
        if scatter is None:
            raise ValueError(f"{op}: weights belong to scattered rows")
        if weights.dtype is not torch.float32:
            raise TypeError(f"{op}: weights must be float32")
        if weights.shape != (R,):
            raise ValueError(f"{op}: weights must be one factor for each of the {R} rows of Y")
    if out is not None:
        if out.dtype is not dtype:
            raise TypeError(f"{op}: out must be {dtype}")
        if out.shape != (R, N) or not out.is_contiguous():
            raise ValueError(f"{op}: out must be dense [{R}, {N}]")
    return R, N, K, E


def run(a: torch.Tensor, sa: torch.Tensor, w: torch.Tensor, sw: torch.Tensor, offsets: torch.Tensor, gather=None,
        topk: int = 1, scatter=None, weights=None, dtype: torch.dtype = torch.bfloat16, out=None, **kwargs):
    global _last_call
    rt.require_device(a, sa, w, sw, offsets, gather, scatter, weights, out)
    R, N, K, E = check(a, sa, w, sw, offsets, gather, topk, scatter, weights, dtype, out)
    Y = a.new_empty((R, N), dtype=dtype) if out is None else out
    if not (R and N):
        return Y
    a, w, offsets = experts.code_rows(a), experts.code_rows(w), offsets.contiguous()
    sa, sa_row, _ = experts.scale_rows(sa)
    sw, sw_row, sw_expert = experts.scale_rows(sw)
    gather = None if gather is None else gather.contiguous()
    scatter = None if scatter is None else scatter.contiguous()
    weights = None if weights is None else weights.contiguous()
    rt.call("tb_moe_mxfp4_grouped_gemm", a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), offsets.data_ptr(),
            rt.ptr(gather), rt.ptr(scatter), rt.ptr(weights), Y.data_ptr(), R, a.shape[0], E, N, K, topk, sa_row, sw_row,
            sw_expert, experts.DTYPES[dtype], rt.stream_handle(a.get_device()))
    _last_call = R, N, K, E
    return Y


def get_last_config():
    return _last_call and {**rt.gemm_tile(rt.OP_MXFP4_GROUPED, *_last_call), "BK": 256}
