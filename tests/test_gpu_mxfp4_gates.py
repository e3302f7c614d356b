"""Gated MXFP4 quantisation where fp32 cannot settle a product: codes and scales are those of silu(gate) * up in 64 bits,
bit for bit, so there is no tolerance."""
import pytest
import torch

from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_torch as quant_ref

pytestmark = pytest.mark.gpu


def check(gate, up):
    from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_hip

    x = torch.cat((gate, up), dim=1)
    codes, scales = impl_hip.run(x.cuda(), gated=True)
    want = quant_ref.run(x, True)
    assert torch.equal(scales.cpu(), want[1])
    assert torch.equal(codes.cpu(), want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("few", [True, False])
def test_gates_below_the_normals(gpu, few, dtype):
    """silu(gate) of such a gate has few bits in fp32; a large up makes an ordinary product of it.  Few: one in 512
    channels, the others 0.75 with an up of 2^-21, whose products are far from every border: nothing else asks for more bits there."""
    print("[gpu case] gates below the normals", few, dtype, flush=True)
    g = torch.Generator().manual_seed(1)
    unit = 2.0 ** (-149 if dtype is torch.float32 else -133)
    M, K = 1000, 512
    gate, up = torch.full((M, K), 0.75), torch.full((M, K), 2.0 ** -21)
    rows = torch.arange(M)
    for at in [torch.randint(0, K, (M,), generator=g)] if few else torch.randperm(K, generator=g)[:200]:
        n = torch.randint(1, 41, (M,), generator=g).float()
        tiny = torch.where(rows % 4 < 2, unit * n, torch.randn(M, generator=g) * 2.0 ** (-125 - 4 * (rows % 4 - 2)))
        # products up to 0.6 * 2^-21, like the others' 0.5 * 2^-21
        u = 1.2 * 2.0 ** -21 * torch.rand(M, generator=g).double() / tiny.double()
        gate[rows, at], up[rows, at] = tiny, u.clamp(-2.0 ** 127, 2.0 ** 127).float()
    gate[0, 0], up[0, 0] = 3 * unit, 2.0 ** 127
    gate, up = gate.to(dtype), up.to(dtype)
    assert bool(torch.isfinite(gate).all() and torch.isfinite(up).all())
    check(gate, up)


def awkward_zeros(rows, K, dtype):
    """Gates and ups with exact zeros of both signs, tokens of zeros alone, and products that vanish in fp32."""
    g = torch.Generator().manual_seed(2)
    gate, up = torch.randn(rows, K, generator=g), torch.randn(rows, K, generator=g)
    for x in (gate, up):
        x[torch.rand(rows, K, generator=g) < 0.02] = 0.0
        x[torch.rand(rows, K, generator=g) < 0.02] = -0.0
    gate[1::4], up[1::8] = -0.0, 0.0
    gate[2::8], up[2::8] = torch.sign(gate[2::8]) * 0.0, torch.sign(up[2::8]) * 0.0
    up[5::16] *= 2.0 ** -120
    gate[5::16] *= 2.0 ** -40
    return gate.to(dtype), up.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_products_of_zeros(gpu, dtype):
    print("[gpu case] gated zeros", dtype, flush=True)
    check(*awkward_zeros(96, 160, dtype))


def test_zeros_are_settled_like_other_products(gpu):
    """Zeros and padded tokens cost no more than other values: a wavefront that goes on to 64 bits takes 2.4 times as
    long, and half of that is allowed.  The least of many timings."""
    print("[gpu case] gated zeros, time", flush=True)
    from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_hip

    def least(x):
        times = []
        for _ in range(30):
            start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(5):
                impl_hip.run(x, gated=True)
            stop.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(stop))
        return min(times)

    M, K = 16384, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(M, 2 * K, generator=g, device="cuda", dtype=torch.bfloat16)
    zeros = x.clone()
    zeros[:, ::50] = -0.0
    padded = x.clone()
    padded[M // 2:] = 0.0
    plain = least(x)
    for name, other in (("zeros", zeros), ("padded", padded)):
        t = least(other)
        print(f"{name}: {t / plain:.2f} of the time", flush=True)
        assert t <= 1.7 * plain
