"""PyTorch reference of paged attention over shared prefixes.

Per sequence: the group's prefix and the own tokens concatenated, scores and
softmax in fp32 (fp64 with dtype=torch.float64), masked after each query's own
position; rows without tokens give 0 and -inf.  Lengths, offsets and page ids
are clamped as the backend clamps them.
"""
import torch


def tokens(cache, scale, ids, length, dtype):
    """[heads, length, D] values of the first `length` tokens on pages `ids`."""
    pages, heads, page, D = cache.shape
    ids = ids.long().clamp(0, pages - 1)
    x = (cache.view(torch.uint8)[ids].view(cache.dtype) if cache.element_size() == 1 else cache[ids]).to(dtype)
    if scale is not None:
        x = x * scale[ids].to(dtype)[..., None]
    return x.transpose(0, 1).reshape(heads, -1, D)[:, :length]


def run(q, k_cache, v_cache, prefix_pages, prefix_lens, group_offsets, pages, lens, cu_q, max_q, scale=None,
        k_scale=None, v_scale=None, dtype=torch.float32, **kwargs):
    T, Hq, D = q.shape
    Hkv, page = k_cache.shape[1:3]
    grp, B, W = Hq // Hkv, *pages.shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=dtype, device=q.device)
    lse = torch.full((T, Hq), -float("inf"), dtype=dtype, device=q.device)
    cu = [min(max(c, 0), T) for c in cu_q.tolist()]
    own = [min(max(n, 0), W * page) for n in lens.tolist()]
    G = 0 if prefix_pages is None else prefix_pages.shape[0]
    bounds = [0] + [min(max(x, 0), B) for x in (group_offsets.tolist()[1:-1] if G else [])] + [B]
    for g in range(max(G, 1)):
        n = min(max(int(prefix_lens[g]), 0), prefix_pages.shape[1] * page) if G else 0
        shared = [tokens(c, s, prefix_pages[g], n, dtype) for c, s in ((k_cache, k_scale), (v_cache, v_scale))] if n \
            else None
        for b in range(bounds[g], bounds[g + 1]):
            n_q = cu[b + 1] - cu[b]
            if n_q <= 0 or n + own[b] == 0:
                continue
            k, v = (tokens(c, s, pages[b], own[b], dtype) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
            if shared:
                k, v = torch.cat((shared[0], k), dim=1), torch.cat((shared[1], v), dim=1)
            x = q[cu[b]:cu[b + 1]].to(dtype).view(n_q, Hkv, grp, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
            s = torch.matmul(x, k.transpose(1, 2).contiguous()).view(Hkv, grp, n_q, -1) * scale
            last = n + own[b] - n_q + torch.arange(n_q, device=q.device)
            hide = torch.arange(k.shape[1], device=q.device) > last[:, None]
            s = s.masked_fill(hide, -float("inf"))
            m = s.amax(dim=-1, keepdim=True)
            p = torch.exp(s - torch.where(m == -float("inf"), torch.zeros_like(m), m)).masked_fill(hide, 0)
            total = p.sum(dim=-1, keepdim=True)
            o = torch.matmul(p.view(Hkv, grp * n_q, -1), v).view(Hkv, grp, n_q, D)
            if not bool(torch.isfinite(v).all()):
                # a value that a row does not attend to leaves no trace in it, not even as 0 * inf
                o = _by_row(p, hide, v)
            o = torch.where(total == 0, torch.zeros_like(o), o / total)
            l = torch.where(total == 0, torch.full_like(m, -float("inf")), m + torch.log(total))
            out[cu[b]:cu[b + 1]] = o.permute(2, 0, 1, 3).reshape(n_q, Hq, D)
            lse[cu[b]:cu[b + 1]] = l[..., 0].permute(2, 0, 1).reshape(n_q, Hq)
    return out.to(q.dtype) if dtype == torch.float32 else out, lse


def _by_row(p, hide, v):
    out = []
    for i in range(hide.shape[0]):
        see = ~hide[i]
        out.append(torch.matmul(p[:, :, i, see], v[:, see]))
    return torch.stack(out, dim=2)
