"""Experts' products on the GPU: segments out of order, a row's bits in the dense and the grouped product, the fresh-input
checks."""
import itertools

import pytest
import torch
import yaml

from tilebench_amd import experts
from tilebench_amd.benchmarks.experts.moe_mxfp4_grouped_gemm import impl_torch as grouped_ref
from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_torch as dequant_ref
from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_torch as quant_ref
from tilebench_amd.data import tensors as T

pytestmark = pytest.mark.gpu


def impl(op):
    import importlib

    return importlib.import_module(f"tilebench_amd.benchmarks.experts.{op}.impl_hip")


def say(*what):
    print("[gpu case]", *what, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def matrix(rows, K, seed):
    return [t.cuda() for t in quant_ref.run(torch.randn(rows, K, generator=gen(seed)))]


def experts_of(E, N, K, seed):
    codes, scales = matrix(E * N, K, seed)
    return codes.view(E, N, -1), experts.empty_scales((E, N), K, "cuda").copy_(scales.view(E, N, -1))


# ----------------------------------------------------------------------------- segments


@pytest.mark.parametrize("R,N,K", [(40, 40, 160), (200, 96, 288), (700, 600, 160)])
def test_segments_out_of_order_write_products_of_their_experts(gpu, R, N, K):
    """Descending and overlapping offsets: what lies around the result stays, and every element is unwritten, or the
    row's product with an expert whose range holds it (columns of a row that several name may come from either)."""
    say("grouped out of order", R, N)
    E = 4
    a, sa = matrix(R, K, 3)
    w, sw = experts_of(E, N, K, 4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    exact = [dequant_ref.values(a, sa) @ dequant_ref.values(w[e], sw[e]).t() for e in range(E)]
    size = [dequant_ref.values(a, sa).abs() @ dequant_ref.values(w[e], sw[e]).abs().t() for e in range(E)]
    for bounds in ((R, 0, R, 0, R), (0, R, 0, R, 0), (R // 2, R, 3, R // 3, R), (-7, R + 9, 5, R + 9, 4), (R, R // 2, 9, 1, 0)):
        room = torch.full((R + 16, N), 7.0, dtype=torch.bfloat16, device="cuda")
        impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, i32(*bounds), out=room[8:8 + R])
        assert bool((room[:8] == 7).all()) and bool((room[8 + R:] == 7).all())
        out = room[8:8 + R].double()
        fits = out == 7
        for e in range(E):
            # one rounding to bf16, and one fp32 step of the magnitudes for every block added
            bound = 2.0 ** -8 * exact[e].abs() + 2.0 ** -134 + (1 + 2.0 ** -7) * 2.0 ** -23 * (K // 32) * size[e]
            m = torch.arange(R, device="cuda")
            held = (m >= max(bounds[e], 0)) & (m < min(bounds[e + 1], R))
            fits |= held[:, None] & ((out - exact[e]).abs() <= bound)
        assert bool(fits.all()), (bounds, int((~fits).sum()))


@pytest.mark.parametrize("R,N,K", [(20, 200, 736), (90, 200, 736), (300, 2000, 2112), (900, 200, 736), (900, 900, 736), (1700, 1304, 1408), (2000, 4096, 4128)])
def test_a_grouped_row_has_the_dense_rows_bits(gpu, R, N, K):
    """Where both calls take mx_tile (which adds the blocks of K in their order, whatever the tile), or both mx_skinny (four
    parts of K in order), a row has the same bits in a dense product, in one expert's segment, and gathered, scattered and
    weighted by 1."""
    say("grouped bits", R, N, K)
    a, sa = matrix(R, K, 3)
    w, sw = experts_of(1, N, K, 4)
    offsets = torch.tensor([0, R], dtype=torch.int32, device="cuda")
    want = impl("mxfp4_gemm").run(a, sa, w[0], sw[0])
    kernel = impl("mxfp4_gemm").get_last_config()["kernel"]
    rows = torch.randperm(R, generator=gen(5)).int().cuda()
    got = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets)
    assert impl("moe_mxfp4_grouped_gemm").get_last_config()["kernel"] == kernel
    assert torch.equal(got, want)
    got = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, gather=rows, scatter=rows, weights=torch.ones(R, device="cuda"))
    assert torch.equal(got, want)


# ----------------------------------------------------------------------------- the harness


@pytest.mark.parametrize("case,dtype", [(dict(tokens=40, topk=4, experts=8, K=736, N=264), torch.bfloat16),
                                        (dict(tokens=300, topk=2, experts=16, K=512, N=384), torch.float16)])
def test_the_grouped_product_passes_the_fresh_input_checks(gpu, case, dtype):
    from tilebench_amd.core.anticache import CHECKS, numerical_checks
    from tilebench_amd.core.verifier import config_per_output, config_tolerance
    from tilebench_amd.paths import operator_config

    op = "moe_mxfp4_grouped_gemm"
    say("anticache", op, case, dtype)
    cfg = yaml.safe_load(open(operator_config(op)))["verify"]
    atol, rtol = config_tolerance(cfg, None)
    seeds = itertools.count(50)

    def make():
        x = T.get_generator(op)(**case, dtype=dtype, seed=next(seeds), device="cpu")
        return tuple(t.to("cuda") if isinstance(t, torch.Tensor) else t for t in x)

    res = numerical_checks(impl(op).run, grouped_ref.run, make, atol=atol, rtol=rtol, per_output=config_per_output(cfg, None))
    assert [r.name for r in res] == list(CHECKS), res[-1].message
    assert all(r.ok for r in res), [r.message for r in res if not r.ok]
    assert not any(r.aliased_inputs or r.mutated_inputs for r in res)
