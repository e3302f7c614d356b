"""hip backend of routing to experts: tb_moe_expert_routing in libtbhip.so.

run(logits [T, E], k) returns (weights float32 [T, k], ids int32 [T, k]).
score "softmax" (over all experts) or "sigmoid" makes scores s of the logits
(float32, float16 or bfloat16); experts are chosen by c = s + bias (float32
[E], None: c = s) and weighted by s.  With groups > 1 (of E / groups consecutive
experts) only the experts of the top_groups groups with the largest group scores,
each the sum of its group_top (1 or 2) largest c, can be chosen.  ids are the k
largest c, descending; equal ones go to the lowest expert, equal groups to the
lowest group.  weights are s of these, divided by their sum if renormalize, times
scale.  Computed in 64 bits and rounded once.
"""
import ctypes

import torch

from tilebench_amd import experts
from tilebench_amd import runtime as rt

rt.load_library()

_last_call = None  # (E, k, groups)
SCORES = ("sigmoid", "softmax")


def check(logits, k, bias=None, groups=1, top_groups=1, group_top=1, score="softmax"):
    """(T, E) of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "moe_expert_routing"
    if logits.dtype not in experts.DTYPES:
        raise TypeError(f"{op}: logits must be float32, float16 or bfloat16")
    if logits.dim() != 2:
        raise ValueError(f"{op}: logits must be [tokens, experts]")
    T, E = logits.shape
    if score not in SCORES:
        raise ValueError(f"{op}: score must be one of {SCORES} (got {score!r})")
    if not 1 <= E <= 1024 or not 1 <= groups <= 64 or E % groups:
        raise ValueError(f"{op}: need 1 to 1024 experts in 1 to 64 groups of equal size (got {E} in {groups})")
    if not 1 <= top_groups <= groups or group_top not in (1, 2) or group_top > E // groups:
        raise ValueError(f"{op}: need 1 to {groups} chosen groups, scored by one or two of their {E // groups} experts "
                         f"(got {top_groups}, {group_top})")
    if not 1 <= k <= min(32, E // groups * top_groups):
        raise ValueError(f"{op}: need 1 <= k <= 32 of the {E // groups * top_groups} experts left (got {k})")
    if bias is not None:
        if bias.dtype is not torch.float32:
            raise TypeError(f"{op}: bias must be float32")
        if bias.shape != (E,):
            raise ValueError(f"{op}: bias must be one value per expert")
    return T, E


def run(logits: torch.Tensor, k: int, bias=None, groups: int = 1, top_groups: int = 1, group_top: int = 1,
        score: str = "softmax", renormalize: bool = True, scale: float = 1.0, **kwargs):
    global _last_call
    rt.require_device(logits, bias)
    T, E = check(logits, k, bias, groups, top_groups, group_top, score)
    weights = logits.new_empty((T, k), dtype=torch.float32)
    ids = logits.new_empty((T, k), dtype=torch.int32)
    if T:
        if E > 1 and logits.stride(1) != 1:
            logits = logits.contiguous()
        bias = None if bias is None else bias.contiguous()
        rt.call("tb_moe_expert_routing", logits.data_ptr(), rt.ptr(bias), weights.data_ptr(), ids.data_ptr(), T, E, k,
                groups, top_groups, group_top, logits.stride(0), score == "softmax", renormalize, scale,
                experts.DTYPES[logits.dtype], rt.stream_handle(logits.get_device()))
    _last_call = E, k, groups
    return weights, ids


def get_last_config():
    if _last_call is None:
        return None
    kernel, lanes, threads = ctypes.c_char_p(), ctypes.c_int32(), ctypes.c_int32()
    rt.call("tb_moe_expert_routing_kernel", *_last_call, *map(ctypes.byref, (kernel, lanes, threads)))
    return {"kernel": kernel.value.decode(), "lanes_per_row": lanes.value, "block": threads.value}
