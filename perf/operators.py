"""Cases of the attention path between a layer's QKV and output projections.

Every case is one pass through one operator, on inputs that already are on
the GPU, over the sizes that serving meets: one token, a decode batch, a
prompt, an image or a video, a batch behind one long system prompt.

kind     operator
rotary   rotary_axes: positions with one to three axes applied to q and k
append   rope_kv_append: q and k rotated, k and v written to a paged cache
attend   shared_prefix_attention: paged attention, shared prefixes read once

``own`` chooses between the plain form (elementary torch operations in 32
bits, angles in 64) and the package's operators.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # an image encoder: 60 x 80 patches, two axes, 80 channels a head, q and k views of one fused projection
        {"name": "rotary_image", "kind": "rotary", "T": 4800, "Hq": 16, "Hk": 16, "D": 80, "R": 80, "axes": 2,
         "interleaved": False, "inverse": False, "dtype": "bf16"},
        # a video prompt: time, height and width over grouped heads
        {"name": "rotary_video", "kind": "rotary", "T": 20001, "Hq": 32, "Hk": 8, "D": 128, "R": 128, "axes": 3,
         "interleaved": False, "inverse": False, "dtype": "fp16"},
        # the gradient of a partial rotation in full precision
        {"name": "rotary_grad", "kind": "rotary", "T": 1500, "Hq": 12, "Hk": 4, "D": 128, "R": 64, "axes": 2,
         "interleaved": True, "inverse": True, "dtype": "fp32"},
        # one decoded token (the smallest call: launch latency)
        {"name": "append_token", "kind": "append", "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "axes": 1, "page": 64,
         "interleaved": False, "dtype": "fp16", "cache": "same"},
        # a decode batch into an 8-bit cache
        {"name": "append_decode_e4m3", "kind": "append", "T": 128, "Hq": 32, "Hkv": 8, "D": 128, "axes": 1, "page": 32,
         "interleaved": False, "dtype": "bf16", "cache": "e4m3"},
        # a long multimodal prompt
        {"name": "append_prompt", "kind": "append", "T": 7001, "Hq": 32, "Hkv": 8, "D": 128, "axes": 3, "page": 64,
         "interleaved": False, "dtype": "bf16", "cache": "same"},
        # a prompt into an 8-bit cache
        {"name": "append_prompt_e4m3", "kind": "append", "T": 4096, "Hq": 32, "Hkv": 8, "D": 128, "axes": 1,
         "page": 64, "interleaved": False, "dtype": "fp16", "cache": "e4m3"},
        # two short conversations of a small model behind a short instruction (latency)
        {"name": "attend_small", "kind": "attend", "B": 2, "q_lo": 1, "q_hi": 1, "Hq": 8, "Hkv": 2, "D": 64, "page": 16,
         "groups": 1, "prefix_lo": 300, "prefix_hi": 300, "own_lo": 5, "own_hi": 40, "dtype": "fp16", "cache": "same"},
        # a decode batch behind one system prompt
        {"name": "attend_decode", "kind": "attend", "B": 64, "q_lo": 1, "q_hi": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "groups": 1, "prefix_lo": 8192, "prefix_hi": 8192, "own_lo": 64, "own_hi": 1024,
         "dtype": "fp16", "cache": "same"},
        # four tenants with prompts of their own, two drafted tokens a step, 8-bit cache
        {"name": "attend_groups_e4m3", "kind": "attend", "B": 96, "q_lo": 1, "q_hi": 2, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 32, "groups": 4, "prefix_lo": 2000, "prefix_hi": 16000, "own_lo": 30, "own_hi": 700,
         "dtype": "bf16", "cache": "e4m3"},
        # eight questions about one very long document
        {"name": "attend_document", "kind": "attend", "B": 8, "q_lo": 1, "q_hi": 1, "Hq": 64, "Hkv": 8, "D": 128,
         "page": 64, "groups": 1, "prefix_lo": 131001, "prefix_hi": 131001, "own_lo": 20, "own_hi": 2000,
         "dtype": "bf16", "cache": "same"},
        # the user's part of sixteen prompts, prefilled behind a cached system prompt
        {"name": "attend_prefill", "kind": "attend", "B": 16, "q_lo": 100, "q_hi": 500, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "groups": 1, "prefix_lo": 6000, "prefix_hi": 6000, "own_lo": 500, "own_hi": 900,
         "dtype": "bf16", "cache": "same"},
    ]


# ----------------------------------------------------------------------------- drawn cases

#: the largest drawn case: bytes of the listed document, operations of the listed prefill
_MOST_BYTES, _MOST_FLOPS, _MOST_TOKENS = 5e8, 3e11, 20000


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "append", "attend", "attend", "attend"])
    if kind == "rotary":
        D = rng.choice([64, 72, 80, 96, 128])
        Hk = rng.choice([1, 2, 4, 8, 16])
        R = D if rng.random() < 0.7 else D // 2
        return {"kind": kind, "T": _log_int(rng, 1, _MOST_TOKENS), "Hq": Hk * rng.choice([1, 2, 4]), "Hk": Hk, "D": D,
                "R": R, "axes": rng.randint(1, 3), "interleaved": rng.random() < 0.4, "inverse": rng.random() < 0.3,
                "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"])}
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 5, 8])
    D, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    dtype, cache = rng.choice(["fp16", "bf16"]), rng.choice(["same", "same", "e4m3"])
    if kind == "append":
        return {"kind": kind, "T": _log_int(rng, 1, 7000), "Hq": Hq, "Hkv": Hkv, "D": D, "axes": rng.randint(1, 3),
                "page": page, "interleaved": rng.random() < 0.3, "dtype": dtype, "cache": cache}
    case = {"kind": kind, "B": _log_int(rng, 1, 128), "q_lo": 1, "q_hi": 1, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "groups": 1, "prefix_lo": 0, "prefix_hi": _log_int(rng, 16, 130000), "own_lo": 1,
            "own_hi": _log_int(rng, 4, 4000), "dtype": dtype, "cache": cache}
    case["groups"] = min(case["B"], rng.choice([1, 1, 1, 2, 5]))
    case["prefix_lo"] = case["prefix_hi"] if case["groups"] == 1 else case["prefix_hi"] // 8
    if rng.random() < 0.35:  # prompts, not tokens
        case["q_hi"] = _log_int(rng, 2, 500)
        case["q_lo"] = max(1, case["q_hi"] // 4)
        case["B"] = max(case["groups"], min(case["B"], 16))
        case["own_lo"], case["own_hi"] = case["q_hi"], max(case["own_hi"], case["q_hi"] + 1)
    while True:
        w = work(dict(case, prefix_lo=case["prefix_hi"], own_lo=case["own_hi"], q_lo=case["q_hi"]))
        if w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS and case["B"] * case["own_hi"] <= 130000:
            return case
        for key, least in (("prefix_hi", 16), ("own_hi", max(4, case["q_hi"] + 1)), ("B", case["groups"])):
            case[key] = max(least, case[key] * 4 // 5)
        case["prefix_lo"] = min(case["prefix_lo"], case["prefix_hi"])


# ----------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _heads(T, counts, D, dtype, g):
    """q, k (, v) as a fused projection leaves them: views of one [T, heads * D] matrix."""
    fused = torch.randn(T, sum(counts) * D, generator=g, device="cuda").to(DTYPES[dtype])
    return [x.view(T, n, D) for n, x in zip(counts, fused.split([n * D for n in counts], dim=1))]


def _frequencies(R, axes, theta):
    """Inverse frequencies of R / 2 pairs and the axis that each pair follows (runs of equal size)."""
    i = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    inv_freq = (theta ** (-2.0 * i / R)).float()
    return inv_freq, (torch.arange(R // 2, device="cuda") * axes // (R // 2)).int()


def _positions(T, axes, g):
    """Text counts up from where the conversation stands; further axes walk a grid of 80 columns."""
    t = torch.arange(T, device="cuda")
    if axes == 1:
        return (t + torch.randint(0, 30000, (1,), generator=g, device="cuda")).int()[None]
    grid = [t // 4800 + torch.randint(0, 3000, (1,), generator=g, device="cuda"), t // 80 % 60, t % 80]
    return torch.stack(grid[-axes:]).int()


def _pool(pages, Hkv, page, D, case, g):
    """k and v caches full of tokens: [pages, Hkv, page, D], and their scales where they are e4m3 codes."""
    out, scales = [], []
    for _ in range(2):
        x = torch.empty((pages, Hkv, page, D), device="cuda", dtype=DTYPES[case["dtype"]])
        x.normal_(generator=g)
        if case["cache"] == "e4m3":
            s = x.abs().amax(dim=-1).float() / 448.0
            x = (x.float() / s[..., None]).to(torch.float8_e4m3fn)
            scales.append(s)
        out.append(x)
    return out + scales


def _spread(n, lo, hi, seed):
    """n whole numbers of lo .. hi, log-uniform, the same on every machine."""
    rng = torch.Generator().manual_seed(1000003 * n + 31 * lo + hi + 7919 * seed)
    u = torch.rand(n, generator=rng).tolist()
    return [max(lo, min(hi, int(round(math.exp(math.log(max(lo, 1)) + x * math.log(max(hi, 1) / max(lo, 1)))))))
            for x in u]


def _lengths(case):
    """Queries, own tokens and prefix lengths of a case, and the sequences of each group."""
    B, G = case["B"], case["groups"]
    n_q = _spread(B, case["q_lo"], case["q_hi"], 1)
    lens = [max(n, x) for n, x in zip(n_q, _spread(B, case["own_lo"], case["own_hi"], 2))]
    prefix = _spread(G, case["prefix_lo"], case["prefix_hi"], 3)
    return n_q, lens, prefix, [B * i // G for i in range(G + 1)]


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, state = _gen(seed), dict(case)
    if case["kind"] == "rotary":
        T, Hq, Hk, D = case["T"], case["Hq"], case["Hk"], case["D"]
        q, k = _heads(T, [Hq, Hk, Hk], D, case["dtype"], g)[:2]
        inv_freq, axes = _frequencies(case["R"], case["axes"], 10000.0)
        return dict(state, x=(q, k, _positions(T, case["axes"], g), inv_freq, axes))
    Hq, Hkv, D, P = case["Hq"], case["Hkv"], case["D"], case["page"]
    if case["kind"] == "append":
        T = case["T"]
        q, k, v = _heads(T, [Hq, Hkv, Hkv], D, case["dtype"], g)
        inv_freq, axes = _frequencies(D, case["axes"], 500000.0)
        # a batch of decoded tokens or a prompt: slots of whole pages, the pages anywhere in the pool
        pages = -(-T // P) + 8
        order = torch.randperm(pages, generator=g, device="cuda")
        if T <= 8 * P:
            slots = torch.randperm(pages * P, generator=g, device="cuda")[:T]
        else:
            t = torch.arange(T, device="cuda") + P // 3
            slots = order[t // P] * P + t % P
        return dict(state, x=(q, k, v, _positions(T, case["axes"], g), inv_freq, axes, slots.int()),
                    cache=_pool(pages, Hkv, P, D, case, g))
    n_q, lens, prefix, bounds = _lengths(case)
    cu = _starts(n_q)
    need = [-(-n // P) for n in prefix], [-(-n // P) for n in lens]
    total = sum(need[0]) + sum(need[1])
    order = torch.randperm(total, generator=g, device="cuda").int()
    tables, at = [], 0
    for counts in need:
        table = torch.zeros((len(counts), max(max(counts), 1)), dtype=torch.int32, device="cuda")
        for i, n in enumerate(counts):
            table[i, :n] = order[at:at + n]
            at += n
        tables.append(table)
    q = (torch.randn(cu[-1], Hq, D, generator=g, device="cuda") * 1.5).to(DTYPES[case["dtype"]])
    return dict(state, q=q, cache=_pool(total, Hkv, P, D, case, g), prefix_pages=tables[0], pages=tables[1],
                prefix_lens=_int32(prefix), lens=_int32(lens), group_offsets=_int32(bounds), cu_q=_int32(cu),
                max_q=max(n_q), plan=(cu, prefix, bounds, max(lens)))


# ----------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "rotary":
        q, k, positions, inv_freq, axes = state["x"]
        cs = _table(positions, inv_freq, axes, state["inverse"])
        return tuple(_rotate(x.float(), cs, state["interleaved"]).to(x.dtype) for x in (q, k))
    return _append(state) if kind == "append" else _attend(state)


def _run_own(state):
    if state["kind"] == "rotary":
        from tilebench_amd.benchmarks.serving.rotary_axes import impl_hip

        return impl_hip.run(*state["x"], interleaved=state["interleaved"], inverse=state["inverse"])
    if state["kind"] == "append":
        from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

        return impl_hip.run(*state["x"], *state["cache"], interleaved=state["interleaved"])
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    k_cache, v_cache, *scales = state["cache"]
    k_scale, v_scale = scales or (None, None)
    return impl_hip.run(state["q"], k_cache, v_cache, state["prefix_pages"], state["prefix_lens"],
                        state["group_offsets"], state["pages"], state["lens"], state["cu_q"], state["max_q"],
                        k_scale=k_scale, v_scale=v_scale)


def _table(positions, inv_freq, axes, inverse=False):
    """cos and sin [T, 1, R / 2] of the angles, the angles themselves in 64 bits."""
    angle = positions.double()[axes.long()].t() * inv_freq.double()
    sin = torch.sin(angle).float()
    return torch.cos(angle).float()[:, None], (-sin if inverse else sin)[:, None]


def _rotate(x, table, interleaved):
    """x fp32 [T, H, D]; the first R channels rotated, the others as they are."""
    cos, sin = table
    P = cos.shape[-1]
    head, tail = x[..., :2 * P], x[..., 2 * P:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :P], head[..., P:])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((head, tail), dim=-1)


def _append(state):
    q, k, v, positions, inv_freq, axes, slots = state["x"]
    k_cache, v_cache, *scales = state["cache"]
    table = _table(positions, inv_freq, axes)
    P = k_cache.shape[2]
    page, at = slots.long() // P, slots.long() % P
    k, v = _rotate(k.float(), table, state["interleaved"]), v.float()
    for i, (x, cache) in enumerate(((k, k_cache), (v, v_cache))):
        if scales:
            s = x.abs().amax(dim=-1) / 448.0
            scales[i][page, :, at] = s
            codes = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x)).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
        else:
            cache[page, :, at] = x.to(cache.dtype)
    return (_rotate(q.float(), table, state["interleaved"]).to(q.dtype), k_cache, v_cache, *scales)


def _gather(state, table):
    """Keys and values of the pages of a table [.., W] as fp32 [.., Hkv, W * P, D]."""
    out = []
    for i in range(2):
        x = state["cache"][i]
        x = (x.view(torch.uint8)[table.long()].view(x.dtype) if x.element_size() == 1 else x[table.long()]).float()
        if len(state["cache"]) == 4:
            x = x * state["cache"][2 + i][table.long()][..., None]
        out.append(x.movedim(-3, -4).flatten(-3, -2))
    return out


def _part(q, k, v, keep, scale):
    """Unnormalised attention over some of the keys: the scores' maximum, the sum and the weighted values."""
    s = (q @ k.transpose(-1, -2)) * scale
    if keep is not None:
        s = torch.where(keep, s, torch.full_like(s, -math.inf))
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return m, p.sum(dim=-1, keepdim=True), p @ v


def _attend(state):
    q, P = state["q"], state["page"]
    T, Hq, D = q.shape
    Hkv, scale = state["Hkv"], 1.0 / math.sqrt(D)
    grp, n, B = Hq // Hkv, state["max_q"], state["B"]
    cu, prefix, bounds, longest = state["plan"]
    rows = q.float().view(T, Hkv, grp, D).transpose(0, 1)                      # [Hkv, T, grp, D]
    # own tokens: all sequences at once, queries and keys padded to the longest
    start, count, lens = state["cu_q"][:-1].long(), state["cu_q"].diff().long(), state["lens"].long()
    i = torch.arange(n, device=q.device)
    at = (start[:, None] + i).clamp(max=T - 1)                                 # [B, n]
    k, v = _gather(state, state["pages"])
    j = torch.arange(k.shape[-2], device=q.device)
    pos = (lens - count)[:, None] + i
    keep = (j <= pos[:, :, None]) & (i < count[:, None])[:, :, None]           # [B, n, L]
    keep = keep[:, None, :, None].expand(B, 1, n, grp, j.numel()).flatten(2, 3)
    qs = rows[:, at].transpose(0, 1).flatten(2, 3)                             # [B, Hkv, n * grp, D]
    parts = [x.view(B, Hkv, n, grp, -1).permute(0, 2, 1, 3, 4) for x in _part(qs, k, v, keep, scale)]
    seq = torch.repeat_interleave(torch.arange(B, device=q.device), count, output_size=T)
    m, l, o = (x[seq, torch.arange(T, device=q.device) - start[seq]] for x in parts)   # [T, Hkv, grp, .]
    # the prefix of each group, once for all its queries
    for g, length in enumerate(prefix):
        a, b = cu[bounds[g]], cu[bounds[g + 1]]
        if length == 0 or a == b:
            continue
        k, v = (x[:, :length] for x in _gather(state, state["prefix_pages"][g, :-(-length // P)]))
        m2, l2, o2 = (x.view(Hkv, b - a, grp, -1).transpose(0, 1)
                      for x in _part(rows[:, a:b].flatten(1, 2), k, v, None, scale))
        top = torch.maximum(m[a:b], m2)
        w1, w2 = torch.exp(m[a:b] - top), torch.exp(m2 - top)
        o[a:b] = o[a:b] * w1 + o2 * w2
        l[a:b] = l[a:b] * w1 + l2 * w2
        m[a:b] = top
    return (o / l).reshape(T, Hq, D).to(q.dtype), (m + torch.log(l)).reshape(T, Hq)


# ----------------------------------------------------------------------------- work


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "rotary":
        T, heads, D, R = case["T"], case["Hq"] + case["Hk"], case["D"], case["R"]
        return {"bytes": 2 * T * heads * D * size + 4 * T * case["axes"] + 4 * R, "flops": 3 * T * heads * R}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    row = D + 4 if case["cache"] == "e4m3" else D * size  # one token of one head of a cache
    if case["kind"] == "append":
        T = case["T"]
        return {"bytes": T * ((2 * Hq + 2 * Hkv) * D * size + 2 * Hkv * row + 4 * case["axes"] + 4) + 4 * D,
                "flops": 3 * T * (Hq + Hkv) * D}
    n_q, lens, prefix, bounds = _lengths(case)
    pairs = 0  # (query, token)
    for g, n in enumerate(prefix):
        for b in range(bounds[g], bounds[g + 1]):
            pairs += n_q[b] * (n + lens[b]) - n_q[b] * (n_q[b] - 1) // 2
    read = sum(prefix) + sum(lens)
    return {"bytes": 2 * read * Hkv * row + sum(n_q) * Hq * (2 * D * size + 4) + 4 * (read // case["page"]),
            "flops": 4 * pairs * Hq * D}


# ----------------------------------------------------------------------------- results in 64 bits


def _turn(x, positions, inv_freq, axes, interleaved, sign=1.0):
    """The rotation as a product of complex numbers."""
    P = inv_freq.numel()
    x = x.double()
    angle = sign * torch.stack([positions[int(a)].double() * f for a, f in zip(axes.tolist(), inv_freq.double())], dim=1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * P].reshape(*x.shape[:2], P, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(*x.shape[:2], 2 * P)
    else:
        z = torch.complex(x[..., :P].contiguous(), x[..., P:2 * P].contiguous()) * turn
        head = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((head, x[..., 2 * P:]), dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        q, k, positions, inv_freq, axes = state["x"]
        sign = -1.0 if case["inverse"] else 1.0
        return tuple(_turn(x, positions, inv_freq, axes, case["interleaved"], sign) for x in (q, k))
    if case["kind"] == "append":
        q, k, v, positions, inv_freq, axes, slots = state["x"]
        P, Hkv, D = case["page"], case["Hkv"], case["D"]
        q, k = (_turn(x, positions, inv_freq, axes, case["interleaved"]) for x in (q, k))
        caches, scales = [], []
        for i, x in enumerate((k, v.double())):
            c = state["cache"][i]
            flat = c.float().double().transpose(1, 2).reshape(-1, Hkv, D)
            if case["cache"] == "e4m3":
                s = x.abs().amax(dim=-1) / 448.0
                whole = state["cache"][2 + i].double().transpose(1, 2).reshape(-1, Hkv)
                scales.append(whole.index_copy(0, slots.long(), s).view(-1, P, Hkv).transpose(1, 2))
                x = (x / s[..., None]).float().to(torch.float8_e4m3fn).float().double()
            caches.append(flat.index_copy(0, slots.long(), x).view(-1, P, Hkv, D).transpose(1, 2))
        return (q, *caches, *scales)
    n_q, lens, prefix, bounds = _lengths(case)
    cu, Hkv, D, P = _starts(n_q), case["Hkv"], case["D"], case["page"]
    grp = case["Hq"] // Hkv

    def tokens(i, table, length):
        """[Hkv, length, D] of cache i, in 64 bits."""
        ids = table[:-(-length // P)].long()
        x = state["cache"][i].view(torch.uint8)[ids].view(state["cache"][i].dtype).double()
        if case["cache"] == "e4m3":
            x = x * state["cache"][2 + i][ids].double()[..., None]
        return x.transpose(0, 1).reshape(Hkv, -1, D)[:, :length]

    out = torch.empty(cu[-1], case["Hq"], D, dtype=torch.float64, device="cuda")
    lse = torch.empty(cu[-1], case["Hq"], dtype=torch.float64, device="cuda")
    for g, length in enumerate(prefix):
        shared = [tokens(i, state["prefix_pages"][g], length) for i in range(2)]
        for b in range(bounds[g], bounds[g + 1]):
            k, v = (torch.cat((shared[i], tokens(i, state["pages"][b], lens[b])), dim=1) for i in range(2))
            q = state["q"][cu[b]:cu[b + 1]].double().view(n_q[b], Hkv, grp, D).permute(1, 2, 0, 3)
            s = (q.reshape(Hkv, -1, D) @ k.transpose(1, 2)).view(Hkv, grp, n_q[b], -1) / math.sqrt(D)
            last = length + lens[b] - n_q[b] + torch.arange(n_q[b], device="cuda")
            s.masked_fill_(torch.arange(k.shape[1], device="cuda") > last[:, None], -math.inf)
            lse[cu[b]:cu[b + 1]] = torch.logsumexp(s, dim=-1).permute(2, 0, 1).reshape(n_q[b], -1)
            o = torch.softmax(s, dim=-1).view(Hkv, grp * n_q[b], -1) @ v
            out[cu[b]:cu[b + 1]] = o.view(Hkv, grp, n_q[b], D).permute(2, 0, 1, 3).reshape(n_q[b], -1, D)
    return out, lse
