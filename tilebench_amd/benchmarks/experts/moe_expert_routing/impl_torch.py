"""PyTorch reference of routing to experts, in 64 bits.

Choices by stable descending sorts, so that equal ones keep the order of their
experts; NaN ranks above every number.
"""
import torch


def scores(x, score):
    x = x.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    top = x.amax(dim=1, keepdim=True)
    p = torch.exp(x - top)
    s = p / p.sum(dim=1, keepdim=True)
    return torch.where(top == -float("inf"), torch.zeros_like(s), s)


def largest(c, n):
    v, i = torch.sort(c, dim=-1, descending=True, stable=True)
    return v[..., :n], i[..., :n]


def run(logits, k, bias=None, groups=1, top_groups=1, group_top=1, score="softmax", renormalize=True, scale=1.0,
        **kwargs):
    T, E = logits.shape
    s = scores(logits, score)
    c = s if bias is None else s + bias.double()
    if groups > 1:
        kept = largest(largest(c.view(T, groups, -1), group_top)[0].sum(dim=-1), top_groups)[1]
        keep = torch.zeros((T, groups), dtype=torch.bool, device=c.device).scatter_(1, kept, True)
        # experts that can be chosen first, each kind in the order of its choices
        keep = keep.repeat_interleave(E // groups, dim=1)
        order = torch.argsort(c, dim=1, descending=True, stable=True)
        order = order.gather(1, torch.argsort(~keep.gather(1, order), dim=1, stable=True))
        ids = order[:, :k]
    else:
        ids = largest(c, k)[1]
    w = s.gather(1, ids)
    if renormalize:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return (w * scale).float(), ids.int()
