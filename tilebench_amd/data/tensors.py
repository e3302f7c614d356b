"""Case-grid expansion and seeded input generators.

Mirrors tilebench/data/tensors.py (``_expand_case_grid:26``, ``expand_cases:610``,
``GENERATORS:560``, ``get_generator:788``, ``infer_problem_size:630``) with one
deliberate change: every generator draws from a seeded CPU ``torch.Generator``
and only then copies to the device, so the CPU oracle, the PyTorch reference
and the GPU backend see identical bytes on any machine (the reference draws
unseeded on the GPU, tensors.py:11, 495-498).
"""
from __future__ import annotations

import math
from itertools import product

import torch

DEFAULT_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cpu").manual_seed(int(seed))


# ----------------------------------------------------------------------------- case grids


_GRID_NAMESPACE = {"__builtins__": {"range": range}, "math": math}


def _normalize_sequence(values, name):
    """The candidates of one grid axis.  An axis is written either as a list or
    as {"expr": "<python expression>"} that evaluates (with range and math
    only) to a list; an empty axis would make an empty grid and is refused."""
    if isinstance(values, dict) and "expr" in values:
        values = eval(values["expr"], dict(_GRID_NAMESPACE))  # noqa: S307 (package configs only)
    if isinstance(values, (list, tuple)) and values:
        return list(values)
    raise ValueError(f"grid axis {name!r}: expected a non-empty list (or an expr giving one), got {values!r}")


def _expand_case_grid(case_grid, case_defaults=None):
    """Every combination of the axes, enumerated with the last YAML key varying
    fastest, each laid over a copy of the defaults."""
    if not isinstance(case_grid, dict) or not case_grid:
        raise ValueError(f"case_grid: expected a mapping of axis name to candidates, got {case_grid!r}")
    names = tuple(case_grid)
    axes = [_normalize_sequence(case_grid[n], n) for n in names]
    base = dict(case_defaults or {})
    return [{**base, **dict(zip(names, values))} for values in product(*axes)]


def expand_cases(operator_name, config):
    """Priority as in the reference: explicit test_cases > case_grid."""
    if config.get("test_cases"):
        defaults = config.get("case_defaults", {})
        return [{**defaults, **c} for c in config["test_cases"]]
    if "case_grid" in config:
        return _expand_case_grid(config["case_grid"], config.get("case_defaults", {}))
    raise ValueError(f"Operator '{operator_name}' config must define test_cases or case_grid.")


# ----------------------------------------------------------------------------- int4 weights


def random_int4_weights(K: int, N: int, group: int, g: torch.Generator, experts: int | None = None):
    """Packed int4 weights with config-0 distributions.

    Codes and zero-points are uniform on [0, 15]; two independent uniform
    nibbles are one uniform byte, so the packed bytes are drawn directly.
    Scales are fp16 uniform on [1e-3, 1e-2].  Returns (packed [.., K, N/2]
    uint8, scales [.., K/G, N] fp16, zeros [.., K/G, N/2] uint8)."""
    if N % 2 or K % group:
        raise ValueError(f"need N even and K % group == 0 (K={K} N={N} group={group})")
    lead = () if experts is None else (experts,)
    packed = torch.randint(0, 256, lead + (K, N // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(lead + (K // group, N), generator=g) * 9e-3 + 1e-3).to(torch.float16)
    zeros = torch.randint(0, 256, lead + (K // group, N // 2), generator=g, dtype=torch.uint8)
    return packed, scales, zeros


def generate_int4_dequant_inputs(K, N, group=128, seed=0, device=DEFAULT_DEVICE, **kwargs):
    """uint8 [K, N/2] packed codes, fp16 scales [K/G, N],
    packed zero-points [K/G, N/2]."""
    packed, scales, zeros = random_int4_weights(K, N, group, _gen(seed))
    return (packed.to(device), scales.to(device), zeros.to(device), int(K), int(N), int(group))


def generate_w4a16_gemm_inputs(M, K, N, group=128, seed=1, device=DEFAULT_DEVICE, layout="rows", **kwargs):
    """fp16 activations [M, K] ~ N(0, 1) and config-0 int4 weights [K, N].

    layout "rows" gives the weights as config 0 packs them (uint8 [K, N/2]);
    "slabs" converts the same weights, on the CPU and before they reach the
    device, to the decode's slab layout (formats.w4a16_to_slabs), a format
    prepared at load time -- only for decode shapes (M <= 16)."""
    if layout not in ("rows", "slabs"):
        raise ValueError(f"unknown W4A16 weight layout {layout!r}")
    if layout == "slabs" and M > 16:
        raise ValueError("the slab layout is a decode format (M <= 16)")
    g = _gen(seed)
    A = torch.randn(M, K, generator=g).to(torch.float16)
    packed, scales, zeros = random_int4_weights(K, N, group, g)
    if layout == "slabs":
        from tilebench_amd.formats import w4a16_to_slabs
        packed = w4a16_to_slabs(packed)
    return (A.to(device), packed.to(device), scales.to(device), zeros.to(device), int(group))


# ----------------------------------------------------------------------------- fp8


def fp8_activations(M, K, outlier_frac=0.001, outlier_scale=20.0, seed=2) -> torch.Tensor:
    """fp16 [M, K] ~ N(0, 1) with round(frac * M * K) entries (a seeded random
    subset) multiplied by `outlier_scale`."""
    g = _gen(seed)
    A = torch.randn(M, K, generator=g)
    n_out = int(round(outlier_frac * M * K))
    if n_out:
        idx = torch.randperm(M * K, generator=g)[:n_out]
        A.view(-1)[idx] *= outlier_scale
    return A.to(torch.float16)


def generate_fp8_act_quant_inputs(M, K, outlier_frac=0.001, outlier_scale=20.0, seed=2,
                                  device=DEFAULT_DEVICE, **kwargs):
    return (fp8_activations(M, K, outlier_frac, outlier_scale, seed).to(device),)


def fp8_weights(K, N, std=0.02, seed=2):
    """Per-column fp8 weights: W ~ N(0, std^2) [K, N], sw[n] = max_k |W[k,n]| / 448,
    Wq = e4m3(W / sw).  Wq is returned as a [K, N] view of an [N, K] row-major
    buffer (K contiguous), the layout torch._scaled_mm takes for its second
    operand (matmul_fp32_fp16_fp8/impl_torch.py:7-18)."""
    g = _gen(seed + 1000)
    W = torch.randn(N, K, generator=g) * std  # stored transposed: row n holds column n of W
    sw = W.abs().amax(dim=1) / 448.0
    Wq_t = (W / sw[:, None]).to(torch.float8_e4m3fn)
    return Wq_t.t(), sw.to(torch.float32)


def generate_fp8_scaled_gemm_inputs(M, N, K, outlier_frac=0.001, outlier_scale=20.0, seed=2,
                                    device=DEFAULT_DEVICE, **kwargs):
    """BASELINE config 2 GEMM operands: (Aq e4m3 [M, K], Wq e4m3 [K, N] K-contiguous,
    sa fp32 [M], sw fp32 [N]); Aq/sa come from the per-token quantiser."""
    from tilebench_amd.benchmarks.operators.fp8_act_quant import impl_torch as quant_ref

    A = fp8_activations(M, K, outlier_frac, outlier_scale, seed)
    Aq, sa = quant_ref.run(A)
    Wq, sw = fp8_weights(K, N, seed=seed)
    return (Aq.to(device), Wq.to(device), sa.to(device), sw.to(device))


def fp8_block_weights(K, N, std=0.02, seed=2, block=128):
    """fp8 weights with one scale per `block` x `block` tile (the layout of
    DeepSeek-V3-style checkpoints): W ~ N(0, std^2) stored as [N, K],
    sw[nb, kb] = max |W over the tile| / 448 (fp32 [ceil(N/block), K/block]),
    WqT = e4m3(W / sw of its tile) [N, K]."""
    if K % block:
        raise ValueError(f"K = {K} is not a multiple of the block size {block}")
    g = _gen(seed + 2000)
    W = torch.randn(N, K, generator=g) * std
    nb = -(-N // block)
    Wp = torch.zeros(nb * block, K)
    Wp[:N] = W
    sw = (Wp.abs().reshape(nb, block, K // block, block).amax(dim=(1, 3)) / 448.0).to(torch.float32)
    s_full = sw.repeat_interleave(block, dim=0)[:N].repeat_interleave(block, dim=1)
    return (W / s_full).to(torch.float8_e4m3fn), sw


def generate_fp8_act_quant_blocks_inputs(M, K, outlier_frac=0.001, outlier_scale=20.0, seed=2,
                                         device=DEFAULT_DEVICE, **kwargs):
    """Config 2a's activations (fp16 with outliers) for the per-token, per-128-channel quantiser."""
    return (fp8_activations(M, K, outlier_frac, outlier_scale, seed).to(device),)


def generate_fp8_block_scaled_gemm_inputs(M, N, K, outlier_frac=0.001, outlier_scale=20.0, seed=2,
                                          device=DEFAULT_DEVICE, **kwargs):
    """Block-scaled fp8 GEMM operands: (Aq e4m3 [M, K], WqT e4m3 [N, K], sa fp32
    [K/128, M], sw fp32 [ceil(N/128), K/128]); Aq/sa from the per-block
    quantiser applied to config 2's activations, the weights from
    fp8_block_weights."""
    from tilebench_amd.benchmarks.operators.fp8_act_quant_blocks import impl_torch as quant_ref

    A = fp8_activations(M, K, outlier_frac, outlier_scale, seed)
    Aq, sa = quant_ref.run(A)
    WqT, sw = fp8_block_weights(K, N, seed=seed)
    return (Aq.to(device), WqT.to(device), sa.to(device), sw.to(device))


# ----------------------------------------------------------------------------- MoE


def generate_moe_topk_gating_inputs(M, E, k, dtype=torch.float32, dist="normal", seed=3,
                                    device=DEFAULT_DEVICE, **kwargs):
    """Router logits [M, E].

    dist="normal": N(0, 1).  dist="grid": every row is a
    seeded permutation of linspace(-3, 3, E), the reference generator's
    distinct-values construction (tensors.py:224-228)."""
    g = _gen(seed)
    if dist == "grid":
        grid = torch.linspace(-3.0, 3.0, steps=E).to(dtype)
        rank = torch.randn(M, E, generator=g).argsort(dim=-1)
        logits = grid[rank]
    elif dist == "normal":
        logits = torch.randn(M, E, generator=g).to(dtype)
    else:
        raise ValueError(f"unknown logits distribution {dist!r}")
    return (logits.to(device), int(M), int(E), int(k))


def zipf_routing(tokens, topk, experts, s=1.1, seed=4):
    """Per token, `topk` distinct experts drawn without replacement with
    probability proportional to rank^-s (rank 1 = most popular), over a seeded
    permutation of the expert ids.  Returns int64 [tokens, topk]."""
    g = _gen(seed)
    perm = torch.randperm(experts, generator=g)
    p = torch.arange(1, experts + 1, dtype=torch.float64).pow(-s)
    p = (p / p.sum()).to(torch.float32)
    ranks = torch.multinomial(p.expand(tokens, experts), topk, replacement=False, generator=g)
    return perm[ranks]


def sorted_padded_layout(choice: torch.Tensor, experts: int, pad: int):
    """Sort (token, slot) pairs by expert (stable) and pad each expert segment to
    a multiple of `pad` rows.  Returns (row_token int64 [R] with -1 on padding
    rows, offsets int32 [E+1], counts int64 [E])."""
    flat = choice.reshape(-1)
    token = torch.arange(choice.shape[0]).repeat_interleave(choice.shape[1])
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=experts)
    padded = (counts + pad - 1) // pad * pad
    offsets = torch.zeros(experts + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(padded, 0)
    row_token = torch.full((int(offsets[-1]),), -1, dtype=torch.int64)
    src = 0
    for e in range(experts):
        n = int(counts[e])
        row_token[offsets[e]:offsets[e] + n] = token[order[src:src + n]]
        src += n
    return row_token, offsets.to(torch.int32), counts


def generate_moe_w4a16_grouped_gemm_inputs(tokens, topk, experts, K, N, group=128, zipf_s=1.1, pad=128,
                                           seed=4, device=DEFAULT_DEVICE, **kwargs):
    """token activations fp16 [tokens, K] ~ N(0, 1) routed to
    `topk` Zipf-distributed experts each, gathered into an expert-sorted,
    per-expert padded buffer A [R, K] (padding rows zero), with per-expert int4
    weights [E, K, N] (config-0 distributions).  Returns (A, packed, scales,
    zeros, offsets int32 [E+1], group)."""
    g = _gen(seed)
    X = torch.randn(tokens, K, generator=g).to(torch.float16)
    choice = zipf_routing(tokens, topk, experts, zipf_s, seed)
    row_token, offsets, _ = sorted_padded_layout(choice, experts, pad)
    A = torch.zeros(row_token.numel(), K, dtype=torch.float16)
    real = row_token >= 0
    A[real] = X[row_token[real]]
    del X
    packed, scales, zeros = random_int4_weights(K, N, group, g, experts=experts)
    return (A.to(device), packed.to(device), scales.to(device), zeros.to(device), offsets.to(device), int(group))


def zipf_router_logits(tokens, experts, s=1.1, g=None):
    """Router logits whose top-k is config 4's routing: log of the Zipf
    popularity rank^-s of each expert (over a seeded permutation of the ids)
    plus standard Gumbel noise, so that the k largest are k distinct experts
    drawn without replacement with probability proportional to popularity.
    fp32 [tokens, experts]."""
    perm = torch.randperm(experts, generator=g)
    rank_of = torch.empty(experts, dtype=torch.int64)
    rank_of[perm] = torch.arange(experts)
    logp = -s * torch.log(rank_of.to(torch.float64) + 1.0)
    u = torch.rand(tokens, experts, generator=g, dtype=torch.float64).clamp_(1e-12, 1.0 - 1e-12)
    return (logp - torch.log(-torch.log(u))).to(torch.float32)


def generate_fused_moe_w4a16_inputs(tokens, experts, topk, H, I, group13=128, group2=64, zipf_s=1.1, seed=15,
                                    device=DEFAULT_DEVICE, **kwargs):
    """MoE layer around config 4: activations X fp16 [tokens, H] ~ N(0, 1),
    router logits fp32 [tokens, E] with config 4's Zipf routing, and per-expert
    int4 weights (config-0 distributions) W13 [E, H, 2I] (gate | up) and W2
    [E, I, H].  Returns (X, logits, W13, S13, Z13, W2, S2, Z2, topk, group13,
    group2)."""
    g = _gen(seed)
    X = torch.randn(tokens, H, generator=g).to(torch.float16)
    logits = zipf_router_logits(tokens, experts, zipf_s, g)
    w13 = random_int4_weights(H, 2 * I, group13, g, experts=experts)
    w2 = random_int4_weights(I, H, group2, g, experts=experts)
    return (X.to(device), logits.to(device), *(t.to(device) for t in w13), *(t.to(device) for t in w2),
            int(topk), int(group13), int(group2))


# ----------------------------------------------------------------------------- reference analog operators


def generate_weight_dequant_inputs(M, TILE_SIZE, dtype=torch.float16, N=None, seed=10, device=DEFAULT_DEVICE,
                                   **kwargs):
    """The reference generator (tensors.py:492-499), seeded: X ~ N(0,1) [M, N],
    S ~ N(0,1) [ceil(M/T), ceil(N/T)], both in `dtype`."""
    N = M if N is None else N
    g = _gen(seed)
    X = torch.randn(M, N, generator=g).to(dtype)
    S = torch.randn(math.ceil(M / TILE_SIZE), math.ceil(N / TILE_SIZE), generator=g).to(dtype)
    return (X.to(device), S.to(device), int(M), int(N), int(TILE_SIZE))


def generate_dequantize_rowwise_inputs(rows, cols, seed=11, device=DEFAULT_DEVICE, **kwargs):
    """The reference generator (tensors.py:179-184), seeded: int8 x in [-128, 127),
    fp32 per-row absmax state in [0, 10)."""
    g = _gen(seed)
    x = torch.randint(-128, 127, (rows, cols), generator=g, dtype=torch.int8)
    state_x = torch.rand(rows, generator=g) * 10.0
    return (x.to(device), state_x.to(device))


def generate_quantize_global_inputs(n, dtype=torch.float32, seed=12, device=DEFAULT_DEVICE, **kwargs):
    """The reference generator (tensors.py:175-176), seeded: fp32 N(0,1) [n]."""
    return (torch.randn(n, generator=_gen(seed)).to(device),)


def generate_matmul_int8_inputs(M, N, K, dtype=torch.int8, seed=13, device=DEFAULT_DEVICE, **kwargs):
    """The reference generator (tensors.py:439-448), seeded: a int8 [M, K] in
    [-64, 64], b uint8 [K/4, N] holding four 2-bit fields per byte."""
    if K % 4:
        raise ValueError("K must be divisible by 4 (B holds 4 fields per byte)")
    g = _gen(seed)
    a = torch.randint(-64, 65, (M, K), generator=g, dtype=torch.int8)
    b = torch.randint(0, 256, (K // 4, N), generator=g, dtype=torch.uint8)
    return (a.to(device), b.to(device))


def generate_matmul_fp32_fp16_fp8_inputs(M, N, K, dtype=torch.float32, seed=14, device=DEFAULT_DEVICE, **kwargs):
    """The reference generator (tensors.py:416-436), seeded: N(0, 1) / sqrt(K)
    operands a [M, K], b [K, N] in `dtype` (fp8 drawn in fp32 and cast)."""
    g = _gen(seed)
    scale = K ** -0.5
    if dtype in (torch.float8_e4m3fn, torch.float8_e5m2):
        a = (torch.randn(M, K, generator=g) * scale).to(dtype)
        b = (torch.randn(K, N, generator=g) * scale).to(dtype)
    else:
        a = (torch.randn(M, K, generator=g) * scale).to(dtype)
        b = (torch.randn(K, N, generator=g) * scale).to(dtype)
    return (a.to(device), b.to(device))


# ----------------------------------------------------------------------------- attention path


def rotary_frequencies(R: int, axes: int, theta: float):
    """Inverse frequencies of R / 2 pairs and the axis each follows (runs of about equal size)."""
    i = torch.arange(R // 2, dtype=torch.float64)
    return (theta ** (-2.0 * i / R)).float(), (torch.arange(R // 2) * axes // (R // 2)).int()


def _rotary_positions(T, axes, g):
    """Text counts up from anywhere; further axes walk the rows of a grid of 60 x 80."""
    t = torch.arange(T) + int(torch.randint(0, 30000, (1,), generator=g)) * (axes == 1)
    return torch.stack([t // 4800, t // 80 % 60, t % 80][-axes:] if axes > 1 else [t]).int()


def _fused_heads(T, counts, D, dtype, g, device):
    """Heads as a fused projection leaves them: views of one [T, heads * D] matrix."""
    fused = torch.randn(T, sum(counts) * D, generator=g).to(dtype).to(device)
    return [x.view(T, n, D) for n, x in zip(counts, fused.split([n * D for n in counts], dim=1))]


def generate_rotary_axes_inputs(T, axes=1, Hq=32, Hk=8, D=128, dtype=torch.float16, seed=0, device=DEFAULT_DEVICE):
    g = _gen(seed)
    q, k, _ = _fused_heads(T, [Hq, Hk, Hk], D, dtype, g, device)
    inv_freq, ax = rotary_frequencies(D, axes, 10000.0)
    return q, k, _rotary_positions(T, axes, g).to(device), inv_freq.to(device), ax.to(device)


def paged_cache(pages, heads, page, D, dtype, g, e4m3=False, device=DEFAULT_DEVICE):
    """k and v pools [pages, heads, page, D] full of N(0, 1) values; e4m3 codes and their scales if asked for."""
    pools = [torch.randn(pages, heads, page, D, generator=g).to(dtype) for _ in range(2)]
    if not e4m3:
        return [x.to(device) for x in pools]
    scales = [x.abs().amax(dim=-1).float() / 448.0 for x in pools]
    pools = [(x.float() / s[..., None]).to(torch.float8_e4m3fn) for x, s in zip(pools, scales)]
    return [x.to(device) for x in pools + scales]


def generate_rope_kv_append_inputs(T, axes=1, Hq=32, Hkv=8, D=128, page=64, cache="same", dtype=torch.float16, seed=0,
                                   device=DEFAULT_DEVICE):
    g = _gen(seed)
    q, k, v = _fused_heads(T, [Hq, Hkv, Hkv], D, dtype, g, device)
    inv_freq, ax = rotary_frequencies(D, axes, 500000.0)
    positions = _rotary_positions(T, axes, g)
    pages = -(-T // page) + 4
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    pools = paged_cache(pages, Hkv, page, D, dtype, g, cache == "e4m3", device)
    return (q, k, v, positions.to(device), inv_freq.to(device), ax.to(device), slots.to(device), *pools)


def generate_shared_prefix_attention_inputs(B, prefix, own, Hq=32, Hkv=8, D=128, page=64, n_q=1, groups=1, cache="same",
                                            dtype=torch.float16, seed=0, device=DEFAULT_DEVICE):
    """B sequences of `own` // 2 .. `own` tokens, n_q queries each, behind `groups` prefixes of `prefix` tokens."""
    g = _gen(seed)
    lens = torch.randint(max(n_q, own // 2), max(n_q, own) + 1, (B,), generator=g).int()
    Wp, W = -(-prefix // page), -(-max(n_q, own) // page)
    order = torch.randperm(groups * Wp + B * W, generator=g).int()
    pools = paged_cache(order.numel(), Hkv, page, D, dtype, g, cache == "e4m3", device)
    q = torch.randn(B * n_q, Hq, D, generator=g).to(dtype)
    bounds = torch.tensor([B * i // groups for i in range(groups + 1)]).int()
    cu_q = (torch.arange(B + 1) * n_q).int()
    shared = (None, None, None) if prefix == 0 else tuple(
        t.to(device) for t in (order[:groups * Wp].view(groups, Wp), torch.full((groups,), prefix).int(), bounds))
    own_pages = order[groups * Wp:].view(B, W)
    return (q.to(device), pools[0], pools[1], *shared, own_pages.to(device), lens.to(device), cu_q.to(device), n_q, None,
            *pools[2:])


GENERATORS = {
    "int4_dequant": generate_int4_dequant_inputs,
    "w4a16_gemm": generate_w4a16_gemm_inputs,
    "fp8_act_quant": generate_fp8_act_quant_inputs,
    "fp8_scaled_gemm": generate_fp8_scaled_gemm_inputs,
    "moe_topk_gating": generate_moe_topk_gating_inputs,
    "moe_w4a16_grouped_gemm": generate_moe_w4a16_grouped_gemm_inputs,
    "weight_dequant": generate_weight_dequant_inputs,
    "dequantize_rowwise": generate_dequantize_rowwise_inputs,
    "quantize_global": generate_quantize_global_inputs,
    "matmul_int8": generate_matmul_int8_inputs,
    "matmul_fp32_fp16_fp8": generate_matmul_fp32_fp16_fp8_inputs,
    "fused_moe_w4a16": generate_fused_moe_w4a16_inputs,
    "fp8_act_quant_blocks": generate_fp8_act_quant_blocks_inputs,
    "fp8_block_scaled_gemm": generate_fp8_block_scaled_gemm_inputs,
    "rotary_axes": generate_rotary_axes_inputs,
    "rope_kv_append": generate_rope_kv_append_inputs,
    "shared_prefix_attention": generate_shared_prefix_attention_inputs,
}


def get_generator(operator_name):
    if operator_name not in GENERATORS:
        raise ValueError(f"No input generator registered for operator: {operator_name}")
    return GENERATORS[operator_name]


def infer_problem_size(operator_name, params):
    """Element count (or 2*M*N*K for GEMMs) of a case, as the reference reports it."""
    p = {k: int(v) for k, v in params.items() if isinstance(v, int)}
    if operator_name == "int4_dequant":
        return p.get("K", 1) * p.get("N", 1)
    if operator_name in ("w4a16_gemm", "fp8_scaled_gemm", "fp8_block_scaled_gemm", "matmul_int8",
                         "matmul_fp32_fp16_fp8"):
        return 2 * p.get("M", 1) * p.get("N", 1) * p.get("K", 1)
    if operator_name in ("fp8_act_quant", "fp8_act_quant_blocks"):
        return p.get("M", 1) * p.get("K", 1)
    if operator_name == "moe_topk_gating":
        return p.get("M", 1) * p.get("E", 1)
    if operator_name == "weight_dequant":
        return p.get("M", 1) * p.get("N", p.get("M", 1))
    if operator_name == "dequantize_rowwise":
        return p.get("rows", 1) * p.get("cols", 1)
    if operator_name == "moe_w4a16_grouped_gemm":
        return 2 * p.get("tokens", 1) * p.get("topk", 1) * p.get("K", 1) * p.get("N", 1)
    if operator_name == "fused_moe_w4a16":
        return 6 * p.get("tokens", 1) * p.get("topk", 1) * p.get("H", 1) * p.get("I", 1)
    if operator_name == "rotary_axes":
        return p.get("T", 1) * (p.get("Hq", 1) + p.get("Hk", 0)) * p.get("D", 1)
    if operator_name == "rope_kv_append":
        return p.get("T", 1) * (p.get("Hq", 1) + 2 * p.get("Hkv", 1)) * p.get("D", 1)
    if operator_name == "shared_prefix_attention":
        return 4 * p.get("B", 1) * p.get("n_q", 1) * (p.get("prefix", 0) + p.get("own", 1)) * p.get("Hq", 1) * p.get("D", 1)
    size, used = 1, False
    for v in p.values():
        size *= max(1, v)
        used = True
    return size if used else 0
