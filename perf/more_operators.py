"""Cases of the microscaled 4-bit (MXFP4) expert layers: routing, quantisation, products.

Every case is one pass through one operator, on inputs that already are on the
GPU, over the sizes that serving meets: one token, a decode batch, a ragged
chunk, a whole prompt.

kind      operator
route     moe_expert_routing: scores, bias for balance, groups, top-k, renormalised weights
quant     mxfp4_quant: activations to e2m1 codes with one power of two for 32 channels, read back as values
dequant   mxfp4_dequant: codes and scales to values
linear    mxfp4_gemm: a linear layer of quantised activations and weights
experts   moe_mxfp4_grouped_gemm: the experts' products over rows sorted by expert

``own`` chooses between the plain form (elementary torch operations in 32
bits; scores and gated activations, whose borders decide, in 64) and the
package's operators.

An MXFP4 matrix [rows, K] is uint8 codes [rows, K / 2], the lower channel in
the low four bits, and uint8 scales [rows, K / 32]: a value is the code's
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit) times 2^(scale - 127).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 32


def listed():
    return [
        # the router of a decode batch: sigmoid scores, a bias for balance, 4 of 8 groups (latency)
        {"name": "route_decode", "kind": "route", "T": 48, "E": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "scale": 2.5, "dtype": "fp32"},
        # the same router over the tokens of long prompts
        {"name": "route_prompt", "kind": "route", "T": 16384, "E": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "scale": 2.5, "dtype": "fp32"},
        # softmax scores over all experts, no groups, 16-bit logits of a ragged batch
        {"name": "route_softmax", "kind": "route", "T": 5001, "E": 60, "k": 4, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_top": 1, "scale": 1.0, "dtype": "bf16"},
        # the input of a linear layer over a prompt
        {"name": "quant_prompt", "kind": "quant", "M": 4096, "K": 7168, "gated": False, "dtype": "bf16"},
        # between the two products of an expert layer: silu(gate) * up of 2001 tokens for 8 experts each
        {"name": "quant_gated", "kind": "quant", "M": 16008, "K": 1408, "gated": True, "dtype": "bf16"},
        # a projection's weights read back for a 16-bit path
        {"name": "dequant_weight", "kind": "dequant", "E": 1, "M": 11008, "K": 4096, "dtype": "bf16"},
        # the weights of a few experts, each with an odd number of blocks a row, in full precision
        {"name": "dequant_experts", "kind": "dequant", "E": 6, "M": 1000, "K": 2912, "dtype": "fp32"},
        # one token through an attention output projection (the smallest product: latency and weights)
        {"name": "linear_token", "kind": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "fp16"},
        # a ragged batch through a narrow projection
        {"name": "linear_batch", "kind": "linear", "M": 200, "N": 2112, "K": 7168, "dtype": "bf16"},
        # a large prefill batch
        {"name": "linear_prompt", "kind": "linear", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16"},
        # gate and up of 64 experts for a decode batch, the tokens' rows gathered
        {"name": "experts_decode", "kind": "experts", "T": 32, "topk": 8, "E": 64, "N": 2816, "K": 4096,
         "step": "up", "dtype": "bf16"},
        # down of 64 experts over a prompt, weighted rows scattered to their tokens
        {"name": "experts_prompt", "kind": "experts", "T": 4096, "topk": 8, "E": 64, "N": 4096, "K": 1408,
         "step": "down", "dtype": "fp16"},
    ]


# ----------------------------------------------------------------------------- drawn cases

#: the largest drawn product and the most bytes, those of the listed ones
_MOST_FLOPS, _MOST_BYTES, _MOST_TOKENS = 1.0e12, 4.0e8, 16384


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "quant", "quant", "dequant", "linear", "linear", "linear", "experts", "experts"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "route":
        E = rng.choice([8, 16, 60, 64, 96, 128, 160, 256, 384])
        groups = rng.choice([n for n in (1, 1, 2, 4, 8, 16) if E % n == 0 and E // n >= 2])
        top = rng.randint((groups + 1) // 2, groups)
        return {"kind": kind, "T": _log_int(rng, 1, _MOST_TOKENS), "E": E, "k": rng.randint(1, min(8, E // groups * top)),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.6, "groups": groups,
                "top_groups": top, "group_top": rng.choice([1, 2]), "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["fp32", "fp32", "fp16", "bf16"])}
    if kind == "quant":
        return {"kind": kind, "M": _log_int(rng, 1, 16384), "K": BLOCK * _log_int(rng, 4, 50),
                "gated": rng.random() < 0.5, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind == "dequant":
        return {"kind": kind, "E": rng.choice([1, 1, 2, 5]), "M": _log_int(rng, 1, 4000), "K": BLOCK * _log_int(rng, 4, 150),
                "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    K = BLOCK * _log_int(rng, 8, 256) if rng.random() < 0.4 else rng.choice([1408, 2048, 4096, 7168, 8192])
    if kind == "linear":
        case = {"kind": kind, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 64, 12288), "K": K, "dtype": dtype}
        if rng.random() < 0.8:
            case["N"] = -(-case["N"] // 16) * 16
        shrink = ("M", "N")
    else:
        E = rng.choice([8, 16, 60, 64])
        case = {"kind": kind, "T": _log_int(rng, 1, 4096), "topk": rng.choice([1, 2, 4, 8]), "E": E,
                "N": 16 * _log_int(rng, 8, 256), "K": min(K, 4096), "step": rng.choice(["up", "down"]), "dtype": dtype}
        shrink = ("T", "N")
    while True:
        w = work(dict(case, T=max(case.get("T", 0), 64)) if kind == "experts" else case)
        if w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS:
            return case
        for key in shrink:
            case[key] = max(1, case[key] * 4 // 5)


# ----------------------------------------------------------------------------- the format, in torch operations


def _scale_values(scales):
    """2^(scale - 127) of uint8 scales in fp32 (255: NaN), from the bits of fp32."""
    s = scales.int()
    bits = torch.where(s == 0, torch.full_like(s, 0x00400000), s << 23)
    return torch.where(s == 255, torch.full_like(s, 0x7FC00000), bits).view(torch.float32)


def _round_e2m1(v):
    """The e2m1 value nearest to every v (ties to the even code, beyond 6: 6)."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _exponents(x):
    """Per block of 32 of x [.., K]: floor(log2(the largest magnitude)) - 2, held to -127 .. 127."""
    top = x.unflatten(-1, (-1, BLOCK)).abs().amax(dim=-1)
    e = torch.frexp(top)[1] - 3
    return torch.where(top == 0, torch.full_like(e, -127), e).clamp(-127, 127)


def _quantise_values(x):
    """x [.., K] as its MXFP4 codes stand for it: fp32 values."""
    e = _exponents(x)
    scale = _scale_values((e + 127).to(torch.uint8))[..., None]
    inverse = _scale_values((127 - e).to(torch.uint8))[..., None].to(x.dtype)
    blocks = x.unflatten(-1, (-1, BLOCK))
    return (_round_e2m1(blocks * inverse).float() * scale).flatten(-2)


def _pack(x):
    """MXFP4 codes and scales of fp32 x [rows, K]; rows of scales start on 16 bytes, as the package's quantiser leaves them."""
    e = _exponents(x)
    q = _round_e2m1(x.unflatten(-1, (-1, BLOCK)) * _scale_values((127 - e).to(torch.uint8))[..., None]).flatten(-2)
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    rows, S = e.shape
    scales = torch.empty((rows, -(-S // 16) * 16), dtype=torch.uint8, device=x.device)[:, :S]
    scales.copy_(e + 127)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _values(codes, scales):
    """fp32 values of codes [.., K / 2] and scales [.., K / 32]."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    m = (code & 7).float()
    a = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))
    a = torch.where(code > 7, -a, a)
    return (a.unflatten(-1, (-1, BLOCK)) * _scale_values(scales)[..., None]).flatten(-2)


# ----------------------------------------------------------------------------- inputs


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, K):
    """N(0, 1) with one channel in a hundred much larger, as a residual stream has them."""
    loud = torch.where(torch.rand(K, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return _randn(g, rows, K) * loud


def _weights(g, rows, K):
    return _pack(_randn(g, rows, K) * 0.02)


def _expert_weights(g, E, N, K):
    """Codes [E, N, K / 2] and scales [E, N, K / 32], one expert at a time."""
    parts = [_weights(g, N, K) for _ in range(E)]
    S = K // BLOCK
    scales = torch.empty((E, N, -(-S // 16) * 16), dtype=torch.uint8, device="cuda")[..., :S]
    for e in range(E):
        scales[e].copy_(parts[e][1])
    return torch.stack([p[0] for p in parts]), scales


def _loads(case, seed):
    """Expert of every (token, slot) pair, popular experts more often: [T, topk] on the host."""
    rng = torch.Generator().manual_seed(7919 + int(seed))
    rank = torch.randperm(case["E"], generator=rng).double() + 1.0
    noise = -torch.log(-torch.log(torch.rand(case["T"], case["E"], generator=rng, dtype=torch.float64).clamp(1e-12, 1 - 1e-12)))
    return torch.topk(noise - 0.7 * torch.log(rank), case["topk"], dim=1).indices


def prepare(case, seed):
    g, state, dtype = torch.Generator(device="cuda").manual_seed(int(seed)), dict(case), DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "route":
        logits = (_randn(g, case["T"], case["E"]) * 1.5).to(dtype)
        bias = _randn(g, case["E"]) * 0.05 if case["bias"] else None
        return dict(state, logits=logits, bias=bias)
    if kind == "quant":
        x = _activations(g, case["M"], case["K"] * (2 if case["gated"] else 1))
        return dict(state, x=x.to(dtype))
    if kind == "dequant":
        codes, scales = _expert_weights(g, case["E"], case["M"], case["K"])
        return dict(state, w=(codes[0], scales[0]) if case["E"] == 1 else (codes, scales))
    N, K = case["N"], case["K"]
    if kind == "linear":
        return dict(state, a=_pack(_activations(g, case["M"], K)), w=_weights(g, N, K))
    T, topk, E = case["T"], case["topk"], case["E"]
    flat = _loads(case, seed).reshape(-1)
    pairs = torch.sort(flat, stable=True).indices
    bounds = [0] + torch.cumsum(torch.bincount(flat, minlength=E), 0).tolist()
    rows = T if case["step"] == "up" else T * topk
    state.update(a=_pack(_activations(g, rows, K)), w=_expert_weights(g, E, N, K), pairs=pairs.int().cuda(),
                 offsets=torch.tensor(bounds, dtype=torch.int32, device="cuda"), plan=bounds)
    if case["step"] == "down":
        weights = torch.rand(T, topk, generator=g, device="cuda") + 0.1
        state["weights"] = (weights / weights.sum(dim=1, keepdim=True)).flatten()
    return state


# ----------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _run_own(state)
    dtype, kind = DTYPES[state["dtype"]], state["kind"]
    if kind == "route":
        return _route(state)
    if kind == "quant":
        return _quantise_values(_gate(state["x"]) if state["gated"] else state["x"].float()).to(dtype)
    if kind == "dequant":
        return _values(*state["w"]).to(dtype)
    if kind == "linear":
        return (_values(*state["a"]) @ _values(*state["w"]).t()).to(dtype)
    return _experts(state, dtype)


def _run_own(state):
    dtype, kind = DTYPES[state["dtype"]], state["kind"]
    if kind == "route":
        from tilebench_amd.benchmarks.experts.moe_expert_routing import impl_hip

        return impl_hip.run(state["logits"], state["k"], state["bias"], groups=state["groups"],
                            top_groups=state["top_groups"], group_top=state["group_top"], score=state["score"],
                            scale=state["scale"])
    if kind in ("quant", "dequant"):
        from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_hip
        from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_hip as quant

        w = quant.run(state["x"], gated=state["gated"]) if kind == "quant" else state["w"]
        return impl_hip.run(*w, dtype=dtype)
    if kind == "linear":
        from tilebench_amd.benchmarks.experts.mxfp4_gemm import impl_hip

        return impl_hip.run(*state["a"], *state["w"], dtype=dtype)
    from tilebench_amd.benchmarks.experts.moe_mxfp4_grouped_gemm import impl_hip

    if state["step"] == "up":
        return impl_hip.run(*state["a"], *state["w"], state["offsets"], gather=state["pairs"], topk=state["topk"],
                            dtype=dtype)
    return impl_hip.run(*state["a"], *state["w"], state["offsets"], scatter=state["pairs"], weights=state["weights"],
                        dtype=dtype)


def _first(x, n):
    """Values and places of the n largest of the last dimension, equal ones in the order of their places."""
    v, i = torch.sort(x, dim=-1, descending=True, stable=True)
    return v[..., :n], i[..., :n]


def _route(state):
    x = state["logits"].double()
    if state["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        p = torch.exp(x - x.amax(dim=1, keepdim=True))
        s = p / p.sum(dim=1, keepdim=True)
    choice = s if state["bias"] is None else s + state["bias"].double()
    T, E = x.shape
    G = state["groups"]
    if G > 1:
        best = _first(choice.view(T, G, E // G), state["group_top"])[0].sum(dim=-1)
        kept = _first(best, state["top_groups"])[1]
        keep = torch.zeros(T, G, dtype=torch.bool, device=x.device)
        keep[torch.arange(T, device=x.device)[:, None], kept] = True
        choice = torch.where(keep.repeat_interleave(E // G, dim=1), choice, torch.full_like(choice, -math.inf))
    ids = _first(choice, state["k"])[1]
    w = s[torch.arange(T, device=x.device)[:, None], ids]
    return (w / w.sum(dim=1, keepdim=True) * state["scale"]).float(), ids.int()


def _gate(x):
    """silu(gate) * up of x [.., 2 K], in 64 bits: a value next to a code's border decides."""
    g, u = x.double().chunk(2, dim=-1)
    return g / (1.0 + torch.exp(-g)) * u


def _experts(state, dtype):
    codes, scales = state["a"]
    w_codes, w_scales = state["w"]
    up, plan = state["step"] == "up", state["plan"]
    pairs = state["pairs"].long()
    a = _values(codes, scales)
    out = torch.empty((pairs.numel(), w_codes.shape[1]), dtype=dtype, device=a.device)
    for e, (lo, hi) in enumerate(zip(plan, plan[1:])):
        if lo == hi:
            continue
        y = (a[pairs[lo:hi] // state["topk"]] if up else a[lo:hi]) @ _values(w_codes[e], w_scales[e]).t()
        if up:
            out[lo:hi] = y.to(dtype)
        else:
            out[pairs[lo:hi]] = (y * state["weights"][pairs[lo:hi]][:, None]).to(dtype)
    return out


# ----------------------------------------------------------------------------- work


def _mx(rows, K):
    return rows * (K // 2 + K // BLOCK)


def work(case):
    kind, size = case["kind"], SIZES[case["dtype"]]
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * size + T * k * 8 + (4 * E if case["bias"] else 0), "flops": T * E * 8}
    if kind == "quant":
        M, K, gated = case["M"], case["K"], case["gated"]
        return {"bytes": M * K * size * (3 if gated else 2) + _mx(M, K), "flops": M * K * (10 if gated else 4)}
    if kind == "dequant":
        rows, K = case["E"] * case["M"], case["K"]
        return {"bytes": _mx(rows, K) + rows * K * size, "flops": rows * K}
    N, K = case["N"], case["K"]
    if kind == "linear":
        M = case["M"]
        return {"bytes": _mx(M + N, K) + M * N * size, "flops": 2 * M * N * K}
    T, pairs, E = case["T"], case["T"] * case["topk"], case["E"]
    # experts that some pair names, the popular ones first: by the loads of one routing
    active = len(set(_loads(case, 0).flatten().tolist()))
    a_rows = T if case["step"] == "up" else pairs
    return {"bytes": _mx(a_rows + active * N, K) + pairs * (N * size + 4 + (4 if case["step"] == "down" else 0)) + 4 * E,
            "flops": 2 * pairs * N * K}


# ----------------------------------------------------------------------------- results in 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _decode(codes, scales):
    """Codes by a table, scales by powers of two, both in 64 bits."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=codes.device)
    out = torch.empty(*codes.shape, 2, dtype=torch.float64, device=codes.device)
    out[..., 0], out[..., 1] = table[(codes % 16).int()], table[(codes // 16).int()]
    power = torch.pow(torch.full((), 2.0, dtype=torch.float64, device=codes.device), scales.double() - 127.0)
    return out.flatten(-2) * power.repeat_interleave(BLOCK, dim=-1)


def _nearest(x):
    """The MXFP4 values of x: codes counted by the borders below a magnitude, ties to even codes."""
    blocks = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    top = blocks.abs().amax(dim=-1, keepdim=True)
    e = torch.floor(torch.log2(top))
    e = e + (torch.pow(2.0, e + 1) <= top).double() - (torch.pow(2.0, e) > top).double()  # log2 next to whole numbers
    unit = torch.pow(2.0, torch.where(top > 0, e - 2.0, torch.full_like(e, -127.0)).clamp(-127, 127))
    a, code = blocks.abs() / unit, 0
    for i in range(7):
        border = (_E2M1[i] + _E2M1[i + 1]) / 2
        code = code + ((a >= border) if i % 2 else (a > border)).int()
    value = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)[code]
    return (torch.sign(blocks) * value * unit).reshape(x.shape)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "route":
        return _exact_route(state)
    if kind == "quant":
        x = state["x"].double()
        if case["gated"]:
            x = x[:, :case["K"]] * torch.special.expit(x[:, :case["K"]]) * x[:, case["K"]:]
        return _nearest(x)
    if kind == "dequant":
        return _decode(*state["w"])
    if kind == "linear":
        return torch.matmul(_decode(*state["a"]), _decode(*state["w"]).t())
    a, (w_codes, w_scales), pairs = _decode(*state["a"]), state["w"], state["pairs"].long()
    out = torch.empty(pairs.numel(), case["N"], dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        lo, hi = state["plan"][e], state["plan"][e + 1]
        w = _decode(w_codes[e], w_scales[e]).t()
        if case["step"] == "up":
            out[lo:hi] = torch.matmul(a[torch.div(pairs[lo:hi], case["topk"], rounding_mode="floor")], w)
        else:
            out[pairs[lo:hi]] = torch.matmul(a[lo:hi], w) * state["weights"].double()[pairs[lo:hi], None]
    return out


def _exact_route(state):
    """Experts taken one at a time: the first of the largest choices left, k times."""
    x, k, G = state["logits"].double(), state["k"], state["groups"]
    s = torch.special.expit(x) if state["score"] == "sigmoid" else torch.softmax(x, dim=1)
    left = s.clone() if state["bias"] is None else s + state["bias"].double()
    T, E = x.shape
    rows = torch.arange(T, device=x.device)
    if G > 1:
        groups = left.view(T, G, E // G)
        best = groups.amax(dim=2)
        if state["group_top"] == 2:
            at = groups.argmax(dim=2, keepdim=True)
            best = best + groups.scatter(2, at, -math.inf).amax(dim=2)
        drop = torch.ones(T, G, dtype=torch.bool, device=x.device)
        for _ in range(state["top_groups"]):
            i = (best == best.amax(dim=1, keepdim=True)).int().argmax(dim=1)
            best[rows, i] = -math.inf
            drop[rows, i] = False
        left = left.masked_fill(drop[:, :, None].expand(T, G, E // G).reshape(T, E), -math.inf)
    ids = torch.empty(T, k, dtype=torch.int32, device=x.device)
    for j in range(k):
        i = (left == left.amax(dim=1, keepdim=True)).int().argmax(dim=1)
        left[rows, i] = -math.inf
        ids[:, j] = i
    w = s.gather(1, ids.long())
    return w * (state["scale"] / w.sum(dim=1, keepdim=True)), ids
