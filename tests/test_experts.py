"""MXFP4 expert layers on the host: the torch references against the formats' and the
routing's definitions in 64 bits, the layouts that are passed on, and what the
operators refuse (checked before any device is touched)."""
import numpy as np
import pytest
import torch
import yaml

from tilebench_amd import experts
from tilebench_amd import runtime as rt
from tilebench_amd.benchmarks.experts.moe_expert_routing import impl_torch as route_ref
from tilebench_amd.benchmarks.experts.moe_mxfp4_grouped_gemm import impl_torch as grouped_ref
from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_torch as dequant_ref
from tilebench_amd.benchmarks.experts.mxfp4_gemm import impl_torch as gemm_ref
from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_torch as quant_ref
from tilebench_amd.core.metrics import work
from tilebench_amd.data import tensors as T
from tilebench_amd.paths import (list_expert_operators, list_operators, list_serving_operators, operator_config,
                                 operator_package)

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def test_operators_are_registered_beside_the_others():
    ops = list_expert_operators()
    assert ops == ["moe_expert_routing", "moe_mxfp4_grouped_gemm", "mxfp4_dequant", "mxfp4_gemm", "mxfp4_quant"]
    assert not set(ops) & (set(list_operators()) | set(list_serving_operators()))
    for op in ops:
        assert operator_package(op) == f"tilebench_amd.benchmarks.experts.{op}"
        cfg = yaml.safe_load(open(operator_config(op)))
        assert T.expand_cases(op, cfg) and T.get_generator(op) is not None


# ----------------------------------------------------------------------------- the format


def nearest(x, gated=False):
    """Codes and scales of rows x, value by value: the code nearest to x / scale, ties to the even code."""
    x = x.double().numpy()
    if gated:
        g, u = np.split(x, 2, axis=-1)
        with np.errstate(over="ignore"):
            x = g / (1 + np.exp(-g)) * u
    rows, K = x.shape
    codes, scales = np.zeros((rows, K), np.uint8), np.zeros((rows, K // 32), np.uint8)
    for r in range(rows):
        for b in range(K // 32):
            block = x[r, 32 * b:32 * b + 32]
            if not np.isfinite(block).all():
                scales[r, b] = 255
                continue
            top = np.abs(block).max()
            e = -127 if top == 0 else min(max(int(np.frexp(top)[1]) - 3, -127), 127)
            scales[r, b] = e + 127
            for i, v in enumerate(block):
                far = np.abs(E2M1 - abs(v) * 2.0 ** -e)
                best = [c for c in range(8) if far[c] == far.min()]
                codes[r, 32 * b + i] = (best[0] if len(best) == 1 else [c for c in best if c % 2 == 0][0]) | \
                    (8 if np.signbit(v) else 0)
    return torch.from_numpy(codes[:, 0::2] | codes[:, 1::2] << 4), torch.from_numpy(scales)


def awkward(rows, K, seed=0):
    """Values over many magnitudes: borders between codes, both zeros, subnormals, the largest, zero blocks, inf and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-140, 120, (rows, 1), generator=g).float())
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 4.0, -0.25, -5.0, 0.0, -0.0])
    x[0] = ties[torch.randint(0, 14, (K,), generator=g)] * 2.0 ** 9
    x[1, :32] = 0
    x[1, 32:] = -0.0
    x[2] = 2.0 ** -149 * torch.randint(-40, 40, (K,), generator=g)
    x[3, 5] = float("inf")
    x[3, 40] = float("nan")
    x[4] = 3.4e38
    return x


def test_quantisation_reference_is_the_definition():
    x = awkward(24, 64)
    want, got = nearest(x), quant_ref.run(x)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0])
    for dtype in (torch.float16, torch.bfloat16):
        x = (torch.randn(5, 96, generator=torch.Generator().manual_seed(1)) * 3).to(dtype)
        assert all(torch.equal(a, b) for a, b in zip(quant_ref.run(x), nearest(x)))
        x = (torch.randn(5, 128, generator=torch.Generator().manual_seed(2)) * 3).to(dtype)
        x[0, :4] = torch.tensor([-90.0, 88.0, -30.0, 0.0])
        assert all(torch.equal(a, b) for a, b in zip(quant_ref.run(x, True), nearest(x, True)))


def test_reading_back_is_the_definition():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, 256)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    got = dequant_ref.values(codes, scales)
    nibble = torch.stack((codes % 16, codes // 16), dim=-1).flatten(1).numpy()
    want = E2M1[nibble % 8] * np.where(nibble > 7, -1, 1)
    with np.errstate(invalid="ignore"):
        want = np.ldexp(want, scales.long().numpy()[:, :1] - 127)
    assert np.array_equal(got[:255].numpy(), want[:255]) and bool(torch.isnan(got[255]).all())
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        assert torch.equal(dequant_ref.run(codes[:255], scales[:255], dtype), got[:255].float().to(dtype))


def test_quantised_values_are_within_half_a_step():
    x = torch.randn(8, 256, generator=torch.Generator().manual_seed(3))
    codes, scales = quant_ref.run(x)
    back = dequant_ref.run(codes, scales, torch.float32).unflatten(-1, (-1, 32))
    scale = torch.exp2(scales.float() - 127)[..., None]
    x = x.unflatten(-1, (-1, 32))
    # steps are scale/2, scale and 2 scale below 2, 4 and 6 of it; beyond 6 (to 8) the value is cut to 6
    bound = torch.where(x.abs() < 2 * scale, 0.25, torch.where(x.abs() < 4 * scale, 0.5, torch.where(x.abs() < 7 * scale, 1.0, 2.0)))
    assert bool(((back - x).abs() <= bound * scale).all())


def test_product_references_agree_with_loops():
    a = T.generate_moe_mxfp4_grouped_gemm_inputs(6, 2, 4, 96, 7, dtype=torch.float16, device="cpu", seed=5)
    codes, scales, w, sw, offsets, pairs, topk = a[:7]
    x, wv = dequant_ref.values(codes, scales), dequant_ref.values(w, sw)
    want = torch.zeros(12, 7, dtype=torch.float64)
    for e in range(4):
        for m in range(int(offsets[e]), int(offsets[e + 1])):
            want[m] = wv[e] @ x[int(pairs[m]) // topk]
    assert torch.equal(grouped_ref.run(*a[:7], dtype=torch.float16, compute=torch.float64), want.half())
    assert torch.equal(gemm_ref.run(codes, scales, w[1], sw[1], torch.float16, torch.float64), (x @ wv[1].t()).half())
    weights = torch.rand(12)
    y = x[pairs.long() // 2]
    b = quant_ref.run(y.float())
    got = grouped_ref.run(*b, w, sw, offsets, scatter=pairs, weights=weights, dtype=torch.float16, compute=torch.float64)
    yv = dequant_ref.values(*b)
    for e in range(4):
        for m in range(int(offsets[e]), int(offsets[e + 1])):
            p = int(pairs[m])
            assert torch.equal(got[p], ((wv[e] @ yv[m]) * weights[p].double()).half())


# ----------------------------------------------------------------------------- routing


def route(row, k, bias, groups, top_groups, group_top, score, renormalize, scale):
    """One row, expert by expert."""
    x = row.double().numpy()
    s = 1 / (1 + np.exp(-x)) if score == "sigmoid" else np.exp(x - x.max()) / np.exp(x - x.max()).sum()
    c = s if bias is None else s + bias.double().numpy()
    per = len(x) // groups
    rank = [-sum(sorted(c[g * per:(g + 1) * per])[-group_top:]) for g in range(groups)]
    kept = sorted(range(groups), key=lambda g: (rank[g], g))[:top_groups] if groups > 1 else [0]
    ids = sorted((e for e in range(len(x)) if e // per in kept), key=lambda e: (-c[e], e))[:k]
    w = s[ids]
    return (w / w.sum() if renormalize else w) * scale, ids


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,k,groups,top_groups,group_top,bias", [
    (16, 4, 1, 1, 1, False), (16, 4, 4, 2, 2, True), (60, 6, 5, 5, 1, True), (12, 2, 6, 1, 2, False), (1, 1, 1, 1, 1, True)])
def test_routing_reference_is_the_definition(score, E, k, groups, top_groups, group_top, bias):
    g = torch.Generator().manual_seed(E + k)
    logits = torch.randn(9, E, generator=g)
    logits[0] = 0.5  # every expert alike: the first ones
    b = torch.randn(E, generator=g) * 0.2 if bias else None
    for renormalize, scale in ((True, 2.5), (False, 1.0)):
        w, ids = route_ref.run(logits, k, b, groups, top_groups, group_top, score, renormalize, scale)
        for t in range(9):
            want = route(logits[t], k, b, groups, top_groups, group_top, score, renormalize, scale)
            assert ids[t].tolist() == want[1]
            np.testing.assert_allclose(w[t].double().numpy(), want[0], rtol=2.0 ** -23, atol=0)
    if not bias:
        assert route_ref.run(logits[:1], k, None, groups, top_groups, group_top, score)[1].tolist() == [list(range(k))]


def test_routing_of_masked_rows():
    inf = float("inf")
    logits = torch.full((4, 8), -inf)
    logits[1, 5] = 0.0
    logits[2, 3] = float("nan")
    w, ids = route_ref.run(logits, 2, score="softmax")
    assert ids[0].tolist() == [0, 1] and w[0].tolist() == [0, 0]
    assert ids[1].tolist() == [5, 0] and w[1].tolist() == [1, 0]
    assert torch.isnan(w[2]).all() and ids[2].tolist() == [0, 1]
    w, ids = route_ref.run(logits, 2, score="sigmoid")
    assert ids[0].tolist() == [0, 1] and w[0].tolist() == [0, 0] and ids[2, 0] == 3
    assert ids[1].tolist() == [5, 0] and w[1].tolist() == [1, 0]


# ----------------------------------------------------------------------------- layouts


def test_rows_of_scales_are_passed_as_they_lie_where_they_can_be():
    s = experts.empty_scales((3, 5), 96 * 32, "cpu")
    assert s.shape == (3, 5, 96) and experts.scale_rows(s) == (s, 96, 480)
    s = experts.empty_scales((5,), 7 * 32, "cpu")
    assert s.stride() == (16, 1) and experts.scale_rows(s)[0] is s and experts.scale_rows(s)[1:] == (16, 80)
    dense = torch.randint(0, 255, (5, 8), dtype=torch.uint8)
    assert experts.scale_rows(dense)[0] is dense and experts.scale_rows(dense)[1] == 8
    for odd in (torch.randint(0, 255, (5, 7), dtype=torch.uint8), dense.t(), dense[:, 1:5], dense[:1].expand(5, 8),
                torch.randint(0, 255, (2, 3, 9), dtype=torch.uint8)):
        got, row, matrix = experts.scale_rows(odd)
        assert torch.equal(got, odd) and row % 4 == 0 and row >= odd.shape[-1] and got.data_ptr() % 4 == 0
        assert got.stride(-2) == row and (odd.dim() == 2 or got.stride(0) == matrix)
    one = torch.zeros(4, 8, dtype=torch.uint8)[:1]  # a row's stride does not matter
    assert experts.scale_rows(one)[1] == 8
    codes = torch.zeros(33, dtype=torch.uint8)[1:].view(2, 16)
    assert experts.code_rows(codes).data_ptr() % 16 == 0


@pytest.mark.parametrize("op,case,dtype,read,written", [
    ("mxfp4_quant", dict(M=6, K=64, gated=False), "fp16", 0, None),
    ("mxfp4_quant", dict(M=6, K=64, gated=True), "bf16", 0, None),
    ("mxfp4_dequant", dict(M=6, K=64), "fp32", None, None)])
def test_configs_count_the_bytes_of_their_tensors(op, case, dtype, read, written):
    from tilebench_amd.core.dtypes import resolve_dtype

    x = T.get_generator(op)(**case, dtype=resolve_dtype(dtype), device="cpu")
    ref = quant_ref if op == "mxfp4_quant" else dequant_ref
    out = ref.run(*x)
    tensors = [t for t in (*x, *(out if isinstance(out, tuple) else (out,))) if isinstance(t, torch.Tensor)]
    assert work(yaml.safe_load(open(operator_config(op)))["metrics"], case, dtype)[1] == \
        sum(t.numel() * t.element_size() for t in tensors)


# ----------------------------------------------------------------------------- refusals


def _impl(op):
    import importlib

    return importlib.import_module(f"tilebench_amd.benchmarks.experts.{op}.impl_hip")


def _mx(*shape):
    return torch.zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8), torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8)


@pytest.mark.parametrize("args,kw,error", [
    ((torch.zeros(4, 64).double(),), {}, TypeError),
    ((torch.zeros(64),), {}, ValueError),
    ((torch.zeros(4, 48),), {}, ValueError),
    ((torch.zeros(4, 0),), {}, ValueError),
    ((torch.zeros(4, 32),), {"gated": True}, ValueError),
    ((torch.zeros(4, 65),), {"gated": True}, ValueError)])
def test_quantisation_refuses(args, kw, error):
    with pytest.raises(error, match="mxfp4_quant"):
        _impl("mxfp4_quant").check(*args, **kw)


@pytest.mark.parametrize("change,error", [
    (lambda x: x.update(codes=x["codes"].int()), TypeError),
    (lambda x: x.update(scales=x["scales"].float()), TypeError),
    (lambda x: x.update(codes=x["codes"][0], scales=x["scales"][0]), ValueError),
    (lambda x: x.update(codes=x["codes"][:, :24], scales=x["scales"]), ValueError),
    (lambda x: x.update(scales=x["scales"][:, :1]), ValueError),
    (lambda x: x.update(scales=x["scales"][:3]), ValueError),
    (lambda x: x.update(dtype=torch.float64), TypeError)])
def test_reading_back_refuses(change, error):
    x = dict(zip(("codes", "scales"), _mx(4, 64)), dtype=torch.float16)
    assert _impl("mxfp4_dequant").check(**x) == 64
    change(x)
    with pytest.raises(error, match="mxfp4_dequant"):
        _impl("mxfp4_dequant").check(**x)


@pytest.mark.parametrize("change,error", [
    (lambda x: x.update(w=_mx(5, 96)[0], sw=_mx(5, 96)[1]), ValueError),
    (lambda x: x.update(w=_mx(2, 5, 64)[0], sw=_mx(2, 5, 64)[1]), ValueError),
    (lambda x: x.update(sa=x["sa"].int()), TypeError),
    (lambda x: x.update(sw=x["sw"].t()), ValueError),
    (lambda x: x.update(dtype=torch.float32), TypeError)])
def test_the_product_refuses(change, error):
    x = dict(zip(("a", "sa", "w", "sw"), (*_mx(4, 64), *_mx(5, 64))))
    assert _impl("mxfp4_gemm").check(**x) == (4, 5, 64)
    change(x)
    with pytest.raises(error, match="mxfp4_gemm"):
        _impl("mxfp4_gemm").check(**x)


@pytest.mark.parametrize("change,error", [
    (lambda x: x.update(offsets=x["offsets"].long()), TypeError),
    (lambda x: x.update(offsets=x["offsets"][:3]), ValueError),
    (lambda x: x.update(gather=torch.zeros(4)), TypeError),
    (lambda x: x.update(gather=torch.zeros(4, 1, dtype=torch.int32)), ValueError),
    (lambda x: x.update(gather=torch.zeros(4, dtype=torch.int32), topk=0), ValueError),
    (lambda x: x.update(gather=torch.zeros(4, dtype=torch.int32), topk=1.0), ValueError),
    (lambda x: x.update(scatter=torch.zeros(3, dtype=torch.int32)), ValueError),
    (lambda x: x.update(weights=torch.zeros(4)), ValueError),
    (lambda x: x.update(scatter=torch.zeros(4, dtype=torch.int32), weights=torch.zeros(4).half()), TypeError),
    (lambda x: x.update(scatter=torch.zeros(4, dtype=torch.int32), weights=torch.zeros(5)), ValueError),
    (lambda x: x.update(out=torch.zeros(4, 5)), TypeError),
    (lambda x: x.update(out=torch.zeros(5, 5).bfloat16()), ValueError),
    (lambda x: x.update(out=torch.zeros(5, 4).bfloat16().t()), ValueError),
    (lambda x: x.update(a=_mx(0, 64)[0], sa=_mx(0, 64)[1], gather=torch.zeros(4, dtype=torch.int32)), ValueError),
    (lambda x: x.update(w=_mx(5, 64)[0], sw=_mx(5, 64)[1]), ValueError),
    (lambda x: x.update(dtype=torch.float32), TypeError)])
def test_the_grouped_product_refuses(change, error):
    x = dict(zip(("a", "sa", "w", "sw"), (*_mx(4, 64), *_mx(3, 5, 64))), offsets=torch.tensor([0, 1, 2, 4]).int())
    assert _impl("moe_mxfp4_grouped_gemm").check(**x) == (4, 5, 64, 3)
    change(x)
    with pytest.raises(error, match="moe_mxfp4_grouped_gemm"):
        _impl("moe_mxfp4_grouped_gemm").check(**x)


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(4, 16).long()), TypeError),
    (dict(logits=torch.zeros(16)), ValueError),
    (dict(logits=torch.zeros(4, 1025)), ValueError),
    (dict(k=0), ValueError), (dict(k=33, logits=torch.zeros(4, 64)), ValueError), (dict(k=17), ValueError),
    (dict(groups=3), ValueError), (dict(groups=0), ValueError), (dict(groups=4, top_groups=5), ValueError),
    (dict(groups=4, top_groups=1, k=5), ValueError), (dict(groups=16, top_groups=4, group_top=2, k=2), ValueError),
    (dict(group_top=3), ValueError), (dict(score="relu"), ValueError),
    (dict(bias=torch.zeros(16).half()), TypeError), (dict(bias=torch.zeros(15)), ValueError)])
def test_routing_refuses(change, error):
    x = dict(logits=torch.zeros(4, 16), k=4)
    assert _impl("moe_expert_routing").check(**x) == (4, 16)
    with pytest.raises(error, match="moe_expert_routing"):
        _impl("moe_expert_routing").check(**dict(x, **change))


def test_steps_between_refuse():
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for bad, error in (((ids.long(), 4), TypeError), ((ids[0], 4), TypeError), ((ids, 0), ValueError), ((ids, 5000), ValueError)):
        with pytest.raises(error, match="align"):
            experts.align(*bad)
    for bad, error in (((torch.zeros(8, 8), ids, 4), TypeError), ((torch.zeros(7, 8).half(), ids, 4), ValueError),
                       ((torch.zeros(8, 8).half(), ids.long(), 4), TypeError)):
        with pytest.raises(error, match="combine"):
            experts.combine(*bad)


def test_the_library_checks_before_it_launches():
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    lib, p = rt.load_library(), 1 << 40  # never dereferenced
    message = lambda: lib.tb_last_error().decode()
    assert lib.tb_mxfp4_quant(None, p, p, 4, 64, 64, 2, 0, 0, None) == rt.TB_E_INVALID and "null" in message()
    assert lib.tb_mxfp4_quant(p, p, p, 4, 48, 64, 2, 0, 0, None) == rt.TB_E_INVALID and "32" in message()
    assert lib.tb_mxfp4_quant(p + 4, p, p, 4, 64, 64, 2, 0, 0, None) == rt.TB_E_ALIGN
    assert lib.tb_mxfp4_quant(p, p, p, 4, 64, 66, 2, 0, 1, None) == rt.TB_E_INVALID and "16 bytes" in message()
    assert lib.tb_mxfp4_quant(p, p, p, 4, 64, 64, 1, 0, 1, None) == rt.TB_E_INVALID and "overlap" in message()
    assert lib.tb_mxfp4_dequant(p, p, p, 4, 64, 2, 3, None) == rt.TB_E_INVALID and "type" in message()
    assert lib.tb_mxfp4_gemm(p, p, p, p, p, 4, 8, 64, 2, 4, 1, None) == rt.TB_E_INVALID and "4 bytes" in message()
    assert lib.tb_mxfp4_gemm(p, p, p, p, p, 4, 8, 64, 4, 4, 0, None) == rt.TB_E_INVALID and "type 0" in message()
    assert lib.tb_mxfp4_gemm(p + 8, p, p, p, p, 4, 8, 64, 4, 4, 1, None) == rt.TB_E_ALIGN
    assert lib.tb_mxfp4_gemm(p, p, p, p, p, 0, 8, 64, 4, 4, 1, None) == rt.TB_E_INVALID
    grouped = lambda **kw: lib.tb_moe_mxfp4_grouped_gemm(*dict(dict(
        a=p, sa=p, w=p, sw=p, offsets=p, gather=None, scatter=None, weights=None, y=p, R=4, a_rows=4, E=2, N=8, K=64,
        topk=1, sa_row=4, sw_row=4, sw_expert=32, dtype=1, stream=None), **kw).values())
    assert grouped(offsets=None) == rt.TB_E_INVALID and "null" in message()
    assert grouped(E=5000) == rt.TB_E_INVALID and "4096" in message()
    assert grouped(a_rows=3) == rt.TB_E_INVALID and "3 rows" in message()
    assert grouped(sw_expert=28) == rt.TB_E_INVALID and "overlap" in message()
    assert grouped(gather=p, a_rows=1 << 26) == rt.TB_E_INVALID and "2 GiB" in message()
    routing = lambda **kw: lib.tb_moe_expert_routing(*dict(dict(
        logits=p, bias=None, weights=p, ids=p, T=4, E=16, k=4, groups=1, top=1, group_top=1, row=16, softmax=0, norm=1,
        scale=1.0, dtype=0, stream=None), **kw).values())
    assert routing(E=1025) == rt.TB_E_INVALID and "1024" in message()
    assert routing(groups=3) == rt.TB_E_INVALID and routing(top=2) == rt.TB_E_INVALID
    assert routing(k=17) == rt.TB_E_INVALID and routing(group_top=3) == rt.TB_E_INVALID
    assert routing(logits=p + 2) == rt.TB_E_ALIGN
