"""Expert layers on the GPU: the steps between the products, references in graphs, a checkpoint's weights."""
import pytest
import torch

from tilebench_amd import experts
from tilebench_amd import formats as F
from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_torch as dequant_ref
from tilebench_amd.benchmarks.experts.mxfp4_gemm import impl_torch as gemm_ref
from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_torch as quant_ref

pytestmark = pytest.mark.gpu


def say(*what):
    print("[gpu case]", *what, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def matrix(rows, K, seed):
    return [t.cuda() for t in quant_ref.run(torch.randn(rows, K, generator=gen(seed)))]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,k,H,skip", [(1, 1, 1, 0), (5, 3, 7, 0), (33, 8, 264, 1), (9, 12, 1030, 3), (0, 2, 7, 0), (4, 2, 0, 0),
                                             (20, 4, 16, 4)])
def test_combine_of_any_rows(gpu, tokens, k, H, skip, dtype):
    """Rows of any length at any address, as the products write them: fp32 additions in slot order, one rounding."""
    say("combine", tokens, k, H, skip, dtype)
    room = torch.randn(tokens * k * H + skip, generator=gen(H)).to(dtype).cuda()
    y = room[skip:].view(tokens * k, H)
    ids = torch.randint(-1, 9, (tokens, k), generator=gen(k)).int()
    total = torch.zeros(tokens, H)
    for j in range(k):
        row = y.cpu().view(tokens, k, H)[:, j].float()
        total = torch.where(((ids[:, j] >= 0) & (ids[:, j] < 8))[:, None], total + row, total)
    got = experts.combine(y, ids.cuda(), 8)
    assert got.shape == (tokens, H) and got.is_contiguous() and torch.equal(got.cpu(), total.to(dtype))


@pytest.mark.parametrize("op", ["mxfp4_dequant", "mxfp4_gemm"])
def test_references_are_captured(gpu, op):
    """A reference that is timed beside a replayed kernel is replayed itself: its graph gives the eager result, again and
    again, on what the inputs hold then."""
    say("reference graph", op)
    a, w = matrix(40, 352, 1), matrix(24, 352, 2)
    args = a if op == "mxfp4_dequant" else (*a, *w)
    ref = dequant_ref if op == "mxfp4_dequant" else gemm_ref
    want = ref.run(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ref.run(*args)
    for i in range(4):
        if i == 2:
            for t, fresh in zip(a, matrix(40, 352, 9)):
                t.copy_(fresh)
            want = ref.run(*args)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(ref.run(*args), want)


@pytest.mark.parametrize("shape", [(40, 2912), (3, 24, 736)])
def test_a_checkpoints_weights_are_laid_out_where_they_are_used(gpu, shape):
    """Rows of scales keep their padding on the GPU, and a product with them is the one with the dense scales."""
    from tilebench_amd.benchmarks.experts.mxfp4_gemm import impl_hip

    say("checkpoint", shape)
    codes, scales = quant_ref.run(torch.randn(shape, generator=gen(1)))
    w = F.mxfp4_checkpoint_to_tb(codes, scales, "cuda")
    assert experts.scale_rows(w.scales)[0] is w.scales and experts.code_rows(w.codes) is w.codes
    assert torch.equal(w.scales.cpu(), scales) and torch.equal(w.codes.cpu(), codes)
    a = matrix(9, shape[-1], 2)
    last = lambda c, s: (c, s) if len(shape) == 2 else (c[-1], s[-1])
    assert torch.equal(impl_hip.run(*a, *last(w.codes, w.scales)), impl_hip.run(*a, *last(codes.cuda(), scales.cuda())))
