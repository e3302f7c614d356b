"""Routing: a row's result is its own, whatever rows lie beside it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def route(*args, **kw):
    from tilebench_amd.benchmarks.experts.moe_expert_routing import impl_hip

    return impl_hip.run(*args, **kw)


@pytest.mark.parametrize("E,k,groups", [(60, 8, 1), (128, 4, 4), (256, 8, 8), (500, 8, 5), (1000, 8, 1)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_rows_beside_odd_ones(gpu, E, k, groups, score):
    """Rows with masked, infinite, huge and missing logits at every place among others: both kinds keep their results."""
    print("[gpu case] routing beside odd rows", E, k, groups, score, flush=True)
    g = torch.Generator().manual_seed(E)
    inf = float("inf")
    logits = torch.randn(70, E, generator=g).cuda() * 2
    bias = (torch.randn(E, generator=g) * 0.1).cuda()
    kw = dict(groups=groups, top_groups=max(1, groups // 2), group_top=2, score=score, scale=2.5)
    plain = route(logits, k, bias, **kw)
    for value in (-inf, inf, float("nan"), 900.0):
        for rows in ([0], [3, 4, 69], list(range(0, 70, 2)), list(range(70))):
            mixed = logits.clone()
            mixed[rows, 1::3] = value
            w, ids = route(mixed, k, bias, **kw)
            rest = [i for i in range(70) if i not in rows]
            assert torch.equal(ids[rest], plain[1][rest]) and torch.equal(w[rest], plain[0][rest])
            for r in rows[:3]:
                alone = route(mixed[r:r + 1], k, bias, **kw)
                assert torch.equal(ids[r], alone[1][0])
                assert torch.equal(w[r].view(torch.int32), alone[0][0].view(torch.int32))


def test_choices_one_step_apart_do_not_depend_on_the_neighbours(gpu):
    """Pairs of neighbouring fp32 logits next to 0, whose scores' difference (2^-30 or so) a bias takes away but for less
    than an fp64 step of the scores: the order within a pair follows the last bits of the exponential, which must not
    change with the rows beside."""
    print("[gpu case] routing pairs", flush=True)
    g = torch.Generator().manual_seed(7)
    for _ in range(600):
        a = -0.01 * torch.arange(1, 5) * (1 + 0.2 * torch.rand(4, generator=g))
        b = torch.nextafter(a, torch.full_like(a, 99.0))
        row = torch.stack((a, b), dim=1).flatten()
        s = torch.sigmoid(row.double())
        bias = torch.zeros(8)
        bias[0::2] = (s[1::2] - s[0::2]).float()
        logits = row.repeat(16, 1)
        logits[13, 4] = 900.0
        w, ids = route(logits.cuda(), 8, bias.cuda(), score="sigmoid", renormalize=False)
        rest = [i for i in range(16) if i != 13]
        assert torch.equal(ids[rest], ids[:1].expand(15, 8)) and torch.equal(w[rest], w[:1].expand(15, 8))
