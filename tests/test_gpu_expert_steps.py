"""Expert layers on the GPU: the steps between the products."""
import pytest
import torch

from tilebench_amd import experts

pytestmark = pytest.mark.gpu


def say(*what):
    print("[gpu case]", *what, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


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
