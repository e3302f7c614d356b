"""PyTorch reference of the experts' MXFP4 products: per expert the gathered rows' values times its weights' values in
fp32 (or the type asked for), weighted and scattered, one rounding.  Rows of Y that nothing goes to are zeros."""
import torch

from tilebench_amd.benchmarks.experts.mxfp4_dequant.impl_torch import values


def run(a, sa, w, sw, offsets, gather=None, topk=1, scatter=None, weights=None, dtype=torch.bfloat16, out=None,
        compute=torch.float32, **kwargs):
    E, N = w.shape[:2]
    x = values(a, sa).to(compute)
    R = x.shape[0] if gather is None else gather.shape[0]
    if gather is not None:
        rows = gather.long() // topk
        seen = (rows >= 0) & (rows < x.shape[0])
        x = torch.where(seen[:, None], x[rows.clamp(0, x.shape[0] - 1)], torch.zeros((), dtype=compute, device=x.device))
    Y = torch.zeros((R, N), dtype=dtype, device=x.device) if out is None else out.clone()
    bounds = [min(max(i, 0), R) for i in offsets.tolist()]
    for e in range(E):
        lo, hi = bounds[e], bounds[e + 1]
        if hi <= lo:
            continue
        y = x[lo:hi] @ values(w[e], sw[e]).to(compute).t()
        if scatter is None:
            Y[lo:hi] = y.to(dtype)
            continue
        at = scatter[lo:hi].long()
        keep = (at >= 0) & (at < R)
        at, y = at[keep], y[keep]
        Y[at] = (y if weights is None else y * weights[at][:, None].to(compute)).to(dtype)
    return Y
