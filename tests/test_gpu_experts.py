"""MXFP4 expert layers on the GPU, against 64-bit references.

Quantised codes and scales, values read back and chosen experts have one right
answer each and are compared bit for bit.  Products: one rounding to 16 bits
(half a step: eps / 2 of the value, half a subnormal step below the normals)
plus the fp32 accumulation, whose error is bounded by one step 2^-23 of the sum
of magnitudes for each of the K / 32 blocks added."""
import pytest
import torch

from tilebench_amd import experts
from tilebench_amd import runtime as rt
from tilebench_amd.benchmarks.experts.moe_expert_routing import impl_torch as route_ref
from tilebench_amd.benchmarks.experts.moe_mxfp4_grouped_gemm import impl_torch as grouped_ref
from tilebench_amd.benchmarks.experts.mxfp4_dequant import impl_torch as dequant_ref
from tilebench_amd.benchmarks.experts.mxfp4_quant import impl_torch as quant_ref
from tilebench_amd.data import tensors as T
from tilebench_amd.data.tensors import mxfp4_matrix

pytestmark = pytest.mark.gpu
HALF = (torch.float16, torch.bfloat16)


def impl(op):
    import importlib

    return importlib.import_module(f"tilebench_amd.benchmarks.experts.{op}.impl_hip")


def say(*what):
    print("[gpu case]", *what, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ----------------------------------------------------------------------------- quantisation


def check_quant(x, gated=False, layout=lambda x: x):
    codes, scales = impl("mxfp4_quant").run(layout(x.cuda()), gated=gated)
    want = quant_ref.run(x, gated)
    assert torch.equal(scales.cpu(), want[1])
    assert torch.equal(codes.cpu(), want[0])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("M,K", [(1, 32), (1, 4096), (3, 96), (37, 1408), (300, 64), (5, 8224), (2, 16416)])
def test_quantisation(gpu, M, K, dtype, gated):
    say("quant", M, K, dtype, gated)
    g = gen(M + K)
    x = torch.randn(M, K * (1 + gated), generator=g) * torch.exp2(torch.randint(-8, 8, (M, 1), generator=g).float())
    x[:, ::7] = 0
    check_quant(x.to(dtype), gated)


@pytest.mark.parametrize("dtype", HALF)
def test_every_16_bit_value_is_quantised(gpu, dtype):
    """All bit patterns in rows of one magnitude, in their order and shuffled, and behind larger values."""
    say("quant every value", dtype)
    v = torch.arange(65536).to(torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    v = torch.cat((v, v[:-v.numel() % 32])).view(-1, 32)
    check_quant(v.clone())
    check_quant(v[:, torch.randperm(32, generator=gen(0))].contiguous().view(-1, 64) if v.shape[0] % 2 == 0 else v)
    for factor in (1.5, 3.0, 11.0, 40.0):
        w = v.clone()
        w[:, 7] = (v.float().abs().amax(dim=1) * factor).clamp(max=float(torch.finfo(dtype).max)).to(dtype)
        check_quant(w)


def test_quantisation_of_awkward_values(gpu):
    from test_experts import awkward

    say("quant awkward")
    check_quant(awkward(40, 256, seed=4))
    x = awkward(6, 64)
    for dtype in HALF:
        y = x.to(dtype)  # the largest overflow to inf
        check_quant(y)
    inf = float("inf")
    g = torch.tensor([[inf, -inf, 0.0, 1.0, -90.0, -104.0, -746.0, 90.0, -1e-30, 3e38, -3e38, float("nan")]]).t()
    u = torch.tensor([1.0, 0.0, -2.0, inf, 3e38, 1e-30])
    x = torch.zeros(g.numel(), u.numel(), 2, 64)
    x[:, :, 0] = torch.linspace(-3, 3, 64)
    x[:, :, 1] = torch.linspace(2, -2, 64)
    x[:, :, 0, 5], x[:, :, 1, 5] = g, u
    check_quant(x.flatten(2).flatten(0, 1), gated=True)
    x[:, :, :, :32] *= torch.tensor([1.0, 1e-36])[None, None, :, None]  # the awkward value decides its block's scale
    x[:, :, 1, 5] = u
    check_quant(x.flatten(2).flatten(0, 1), gated=True)


def test_gated_values_next_to_borders_fall_on_the_right_side(gpu):
    """up chosen so that silu(gate) * up lies within a rounding of a border between two codes or two scales."""
    say("quant gated borders")
    g = gen(9)
    gate = torch.rand(4096, 32, generator=g) * 6 + 0.25
    silu = gate.double() / (1 + torch.exp(-gate.double()))
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 2.0, 8.0])[torch.randint(0, 10, (4096, 32), generator=g)]
    up = (border.double() / silu).float()
    up[::2] = torch.nextafter(up[::2], torch.full_like(up[::2], 100.0))
    up[1::4, 3:] = 0.01  # one value decides the scale
    check_quant(torch.cat((gate, up), dim=1), gated=True)


def test_quantisation_takes_any_strides(gpu):
    say("quant strides")
    g = gen(3)
    x = torch.randn(6, 5, 192, generator=g).half()
    for layout in (lambda x: x, lambda x: x.transpose(0, 1), lambda x: x[:, 1:3], lambda x: x[..., 32:96],
                   lambda x: x[..., 3:99], lambda x: x[:1].expand(4, 5, 192), lambda x: x[0].t().contiguous().t(),
                   lambda x: x[:0]):
        view = layout(x)
        codes, scales = impl("mxfp4_quant").run(layout(x.cuda()))
        want = quant_ref.run(view)
        assert codes.shape == want[0].shape and torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
        assert scales.numel() == 0 or scales.data_ptr() % 4 == 0


# ----------------------------------------------------------------------------- reading back


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
def test_every_code_and_scale_reads_back(gpu, dtype):
    say("dequant every code", dtype)
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    got, want = impl("mxfp4_dequant").run(codes.cuda(), scales.cuda(), dtype).cpu(), dequant_ref.run(codes, scales, dtype)
    assert bool(torch.isnan(got[255]).all()) and torch.equal(got[:255], want[:255])


@pytest.mark.parametrize("shape", [(1, 32), (7, 2912), (3, 5, 96), (2, 3, 4, 64), (0, 64), (1, 16416)])
def test_reading_back_takes_any_shape(gpu, shape):
    say("dequant", shape)
    x = torch.randn(shape, generator=gen(1))
    codes, scales = mxfp4_matrix(x, "cpu")
    want = dequant_ref.run(codes, scales)
    for s in (scales, scales.contiguous()):
        assert torch.equal(impl("mxfp4_dequant").run(codes.cuda(), s.cuda()).cpu(), want)
    if len(shape) == 3:
        got = impl("mxfp4_dequant").run(codes.cuda().transpose(0, 1), scales.cuda().transpose(0, 1))
        assert torch.equal(got.cpu(), want.transpose(0, 1))


# ----------------------------------------------------------------------------- products


def matrix(rows, K, seed, spread=0):
    g = gen(seed)
    x = torch.randn(rows, K, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-spread, spread + 1, (rows, K // 32), generator=g).float()).repeat_interleave(32, 1)
    return [t.cuda() for t in quant_ref.run(x)]


def check_close(got, exact, magnitude, K):
    """got against the fp64 product `exact`; magnitude: the products' magnitudes added up."""
    t = torch.finfo(got.dtype)
    bound = t.eps / 2 * exact.abs() + t.smallest_normal * t.eps / 2 + (1 + t.eps) * 2.0 ** -23 * (K // 32) * magnitude
    off = (got.double() - exact).abs()
    assert bool((off <= bound).all()), f"{int((off > bound).sum())} of {off.numel()} off, most {float((off / bound).max()):.3g} of the bound"


def check_gemm(a, sa, w, sw, dtype, K, out=None):
    got = impl("mxfp4_gemm").run(a, sa, w, sw, dtype)
    x, v = dequant_ref.values(a, sa), dequant_ref.values(w, sw)
    check_close(got, x @ v.t(), x.abs() @ v.abs().t(), K)
    return got


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 32), (1, 4096, 4096), (2, 33, 64), (17, 130, 96), (31, 31, 224), (32, 32, 256), (33, 63, 288), (32, 96, 1024),
    (64, 64, 512), (65, 65, 544), (100, 200, 2080), (129, 257, 160), (200, 2112, 736), (16, 1000, 7168), (48, 72, 8192)])
def test_product(gpu, M, N, K, dtype):
    say("gemm", M, N, K, dtype)
    check_gemm(*matrix(M, K, M), *matrix(N, K, N + 1), dtype, K)


@pytest.mark.parametrize("M,N,K,tile", [
    (700, 700, 544, 32), (1700, 1900, 96, 64), (200, 2112, 7168, 64), (260, 4097, 4128, 64), (3500, 3600, 96, 128),
    (1801, 8193, 1056, 128), (4001, 4001, 1056, 128), (4001, 8001, 512, 128), (2500, 6000, 2080, 256), (4001, 4004, 2080, 256), (2500, 6001, 2112, 256),
    (2500, 6001, 4160, 256), (2600, 5504, 4128, 256), (1801, 2001, 4128, 128), (700, 3000, 2080, 128), (300, 7999, 2336, 128),
    (2048, 2048, 8192, 128), (2048, 4001, 4128, 256), (1500, 4104, 2336, 256), (2007, 3100, 8192, 256)])
def test_product_on_every_tile(gpu, M, N, K, tile):
    say("gemm", M, N, K)
    picked = rt.gemm_tile(rt.OP_MXFP4, M, N, K)
    assert picked["BM"] == tile
    assert picked["waves"] == (8 if tile == 256 and (K <= 4096 or picked["BN"] == 128) else 4)
    check_gemm(*matrix(M, K, 1), *matrix(N, K, 2), torch.bfloat16, K)


def test_product_of_blocks_of_different_scales(gpu):
    say("gemm spread")
    for M in (5, 70):
        check_gemm(*matrix(M, 512, 3, 12), *matrix(80, 512, 4, 12), torch.bfloat16, 512)
        check_gemm(*matrix(M, 480, 3, 3), *matrix(80, 480, 4, 3), torch.float16, 480)


@pytest.mark.parametrize("M", [3, 70, 1500])
@pytest.mark.parametrize("K", [32, 224, 512])
def test_nothing_behind_the_last_channel_counts(gpu, M, K):
    """Operands as the head of wider rows: codes behind K, and scales of NaN and the largest power, leave no trace."""
    say("gemm tail", M, K)
    N = 1600 if M > 1000 else 40
    a, sa = matrix(M, K, 5)
    w, sw = matrix(N, K, 6)
    wide = []
    for s in (sa, sw):
        t = torch.full((s.shape[0] + 1, -(-s.shape[1] // 16) * 16 + 16), 255, dtype=torch.uint8, device="cuda")
        t[:, ::2] = 254
        t[:-1, :s.shape[1]] = s
        wide.append(t[:-1, :s.shape[1]])
    codes = []
    for c in (a, w):
        t = torch.full((c.shape[0] + 1, c.shape[1]), 0x77, dtype=torch.uint8, device="cuda")
        t[:-1] = c
        codes.append(t[:-1])
    got = impl("mxfp4_gemm").run(codes[0], wide[0], codes[1], wide[1])
    assert torch.equal(got, check_gemm(a, sa, w, sw, torch.bfloat16, K))


@pytest.mark.parametrize("M", [4, 90])
def test_extreme_scales(gpu, M):
    say("gemm scales", M)
    K = 128
    a, sa = matrix(M, K, 7)
    w, sw = matrix(48, K, 8)
    clean = impl("mxfp4_gemm").run(a, sa, w, sw)
    for where in (0, 2, 3):
        s = sa.clone()
        s[1, where] = 255
        got = impl("mxfp4_gemm").run(a, s, w, sw)
        assert bool(torch.isnan(got[1]).all())
        assert torch.equal(got[torch.arange(M) != 1], clean[torch.arange(M) != 1])
        s = sw.clone()
        s[9, where] = 255
        got = impl("mxfp4_gemm").run(a, sa, w, s)
        assert bool(torch.isnan(got[:, 9]).all()) and torch.equal(got[:, :9], clean[:, :9])
    # the smallest scale times the largest is 1; the smallest squared is nothing
    small, large = torch.zeros_like(sa), torch.full_like(sw, 254)
    one = (torch.full_like(sa, 127), torch.full_like(sw, 127))
    assert torch.equal(impl("mxfp4_gemm").run(a, small, w, large), impl("mxfp4_gemm").run(a, one[0], w, one[1]))
    assert not bool(impl("mxfp4_gemm").run(a, small, w, torch.zeros_like(sw)).any())


def test_product_takes_any_layout(gpu):
    say("gemm layouts")
    a, sa = matrix(40, 352, 1)
    w, sw = matrix(24, 352, 2)
    want = impl("mxfp4_gemm").run(a, sa, w, sw)
    again = [torch.cat((t[:, :3], t), dim=1)[:, 3:] for t in (a, sa, w, sw)]          # odd addresses and strides
    assert torch.equal(impl("mxfp4_gemm").run(*again), want)
    again = [t.t().contiguous().t() for t in (a, sa, w, sw)]
    assert torch.equal(impl("mxfp4_gemm").run(*again), want)
    for m, n in ((0, 24), (40, 0), (1, 24), (40, 1)):
        got = impl("mxfp4_gemm").run(a[:m], sa[:m], w[:n], sw[:n])
        assert got.shape == (m, n)
        check_close(got, want[:m, :n].double(), want[:m, :n].double().abs(), 352)


def check_grouped(a, sa, w, sw, offsets, dtype, K, **kw):
    R, N = (a.shape[0] if kw.get("gather") is None else kw["gather"].shape[0]), w.shape[1]
    mark = torch.full((R, N), 7.0, dtype=dtype, device="cuda")
    got = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, dtype=dtype, out=mark.clone(), **kw)
    exact = grouped_ref.run(a, sa, w, sw, offsets, dtype=torch.float64, out=mark.double(), compute=torch.float64, **kw)
    sign = torch.full_like(a, 0x77)  # codes without their signs
    size = grouped_ref.run(a & sign, sa, w & 0x77, sw, offsets, dtype=torch.float64, out=torch.zeros_like(exact),
                           compute=torch.float64, **kw)
    check_close(got, exact, size, K)
    return got


def experts_of(E, N, K, seed):
    codes, scales = matrix(E * N, K, seed)
    return codes.view(E, N, -1), experts.empty_scales((E, N), K, "cuda").copy_(scales.view(E, N, -1))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("counts,N,K", [
    ([1], 8, 32), ([3, 0, 1], 40, 96), ([0, 0, 5, 0], 33, 256), ([30, 33, 64, 1, 0, 7], 72, 1408),
    ([200, 0, 3, 129], 136, 544), ([1] * 70, 64, 288), ([0] * 130 + [40], 48, 64)])
def test_grouped_product(gpu, counts, N, K, dtype):
    say("grouped", counts, N, K, dtype)
    R, E = sum(counts), len(counts)
    a, sa = matrix(R, K, R)
    w, sw = experts_of(E, N, K, E + 1)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    plain = check_grouped(a, sa, w, sw, offsets, dtype, K)
    g = gen(K)
    gather = torch.randint(0, 3 * R, (R,), generator=g).int().cuda()
    check_grouped(a, sa, w, sw, offsets, dtype, K, gather=gather, topk=3)
    scatter = torch.randperm(R, generator=g).int().cuda()
    check_grouped(a, sa, w, sw, offsets, dtype, K, scatter=scatter, weights=torch.rand(R, generator=g).cuda())
    assert torch.equal(check_grouped(a, sa, w, sw, offsets, dtype, K, scatter=scatter)[scatter.long()], plain)


@pytest.mark.parametrize("rows,N,K,tile", [
    (20, 600, 288, (32, 32)), (330, 900, 96, (32, 128)), (50, 640, 1408, (32, 128)), (700, 600, 160, (32, 128)),
    (6, 2815, 4128, (64, 64)), (1400, 1300, 96, (128, 128)), (600, 1200, 544, (128, 128)), (1400, 1304, 1408, (256, 256)),
    (2000, 2001, 1056, (256, 256)), (330, 900, 1408, (128, 128)), (400, 1000, 2336, (128, 128)), (330, 1899, 4128, (256, 128)),
    (700, 1200, 2080, (256, 128))])
def test_grouped_product_on_every_tile(gpu, rows, N, K, tile):
    say("grouped", rows, N, K)
    counts = [rows, rows // 3, 0, rows * 2, rows - 1, 300, 257, rows + 5] if rows > 6 else [rows, 3, 0, 65, 1, 20, 4, 1]
    R, E = sum(counts), len(counts)
    picked = rt.gemm_tile(rt.OP_MXFP4_GROUPED, R, N, K, E)
    assert (picked["BM"], picked["BN"]) == tile
    a, sa = matrix(R, K, 3)
    w, sw = experts_of(E, N, K, 4)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    check_grouped(a, sa, w, sw, offsets, torch.bfloat16, K)
    g = gen(K)
    check_grouped(a, sa, w, sw, offsets, torch.float16, K, gather=torch.randint(0, 2 * R, (R,), generator=g).int().cuda(),
                  topk=2, scatter=torch.randperm(R, generator=g).int().cuda(), weights=torch.rand(R, generator=g).cuda())


@pytest.mark.parametrize("R,N", [(40, 40), (700, 600)])
def test_rows_outside_every_segment_are_left_alone(gpu, R, N):
    """Offsets that start late and end early, rows to gather and to write that do not exist, offsets out of range and out
    of order: nothing but the named rows is written, and nothing outside is read."""
    say("grouped rows", R, N)
    K, E, n = 160, 4, R // 4
    a, sa = matrix(R, K, 3)
    w, sw = experts_of(E, N, K, 4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for offsets in (i32(2, n, n, 2 * n, 3 * n), i32(0, 0, 0, 0, 0), i32(-5, n, 2 * n, 3 * n, R + 1000),
                    i32(0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1), i32(R, R, R, R, R)):
        check_grouped(a, sa, w, sw, offsets, torch.bfloat16, K)
    offsets = i32(0, n, 2 * n, 3 * n, R)
    g = gen(1)
    gather = torch.randint(-R, 2 * R, (R,), generator=g).int().cuda()
    gather[3], gather[7] = 2 ** 31 - 1, -2 ** 31
    check_grouped(a, sa, w, sw, offsets, torch.bfloat16, K, gather=gather)
    scatter = torch.randperm(2 * R, generator=g)[:R].int().cuda() - 5
    scatter[3], scatter[7] = 2 ** 31 - 1, -2 ** 31
    check_grouped(a, sa, w, sw, offsets, torch.bfloat16, K, scatter=scatter, weights=torch.rand(R, generator=g).cuda())
    # descending offsets: whatever they name, the call ends and writes no row twice as long as it is
    out = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, i32(R, 0, R, 0, R))
    torch.cuda.synchronize()
    assert out.shape == (R, N)


def test_a_grouped_row_is_the_dense_row(gpu):
    """One expert of many rows gives the dense product's rows; weights of 1 change nothing."""
    say("grouped against dense")
    K, N = 736, 200
    for R in (20, 90, 900):
        a, sa = matrix(R, K, 3)
        w, sw = experts_of(1, N, K, 4)
        offsets = torch.tensor([0, R], dtype=torch.int32, device="cuda")
        rows = torch.arange(R, device="cuda").int()
        want = impl("mxfp4_gemm").run(a, sa, w[0], sw[0])
        got = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, gather=rows, scatter=rows,
                                                 weights=torch.ones(R, device="cuda"))
        check_close(got, want.double(), want.double().abs(), K)


@pytest.mark.parametrize("R,N", [(50, 72), (700, 600)])
def test_a_row_named_twice_holds_values_of_either(gpu, R, N):
    say("grouped twice", R, N)
    a, sa = matrix(R, 160, 1)
    w, sw = experts_of(3, N, 160, 2)
    offsets = torch.tensor([0, R // 3, R // 2, R], dtype=torch.int32, device="cuda")
    plain = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets)
    scatter = torch.arange(R, dtype=torch.int32, device="cuda")
    scatter[R - 1] = 2                                    # rows 2 and R - 1 both go to 2, none to R - 1
    out = torch.full_like(plain, 7.0)
    impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, scatter=scatter, out=out)
    assert bool(((out[2] == plain[2]) | (out[2] == plain[R - 1])).all()) and bool((out[R - 1] == 7).all())
    rest = torch.arange(R - 1, device="cuda") != 2
    assert torch.equal(out[:-1][rest], plain[:-1][rest])


@pytest.mark.parametrize("R,N,K", [(40, 64, 96), (700, 600, 160), (1500, 2048, 1056)])
def test_results_at_odd_addresses(gpu, R, N, K):
    say("grouped odd addresses", R, N)
    a, sa = matrix(R, K, 1)
    w, sw = experts_of(3, N, K, 2)
    index = torch.stack((torch.arange(R).flip(0), torch.arange(R)), dim=1).int().cuda()[:, 0]        # a stride of 2
    factors = torch.rand(R, 2, generator=gen(3)).cuda()[:, 1]
    offsets = torch.tensor([0, 9, R // 2, 9, R // 2, 9, R, 9], dtype=torch.int32, device="cuda")[::2]
    kw = dict(scatter=index, weights=factors)
    want = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, **kw)
    room = torch.full((R * N + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[3:3 + R * N].view(R, N)
    assert impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, offsets, out=out, **kw) is out
    assert torch.equal(out, want) and bool((room[:3] == 7).all()) and bool((room[3 + R * N:] == 7).all())


@pytest.mark.parametrize("R", [3, 300])
def test_thousands_of_experts(gpu, R):
    """Every segment is looked up among all experts: the first, the last and one in between have rows."""
    say("grouped experts", R)
    E, N, K = 4096, 40, 64
    w, sw = experts_of(E, N, K, 3)
    a, sa = matrix(R, K, 4)
    counts = torch.zeros(E, dtype=torch.int64)
    counts[0], counts[2111], counts[E - 1] = 1, 1, R - 2
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), counts.cumsum(0))).int().cuda()
    check_grouped(a, sa, w, sw, offsets, torch.bfloat16, K)


def random_bytes(lo, hi, *shape):
    return torch.randint(lo, hi, shape, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("R", [3, 300])
def test_weights_behind_4_gib(gpu, R):
    say("grouped far weights", R)
    E, N, K = 6, 1 << 18, 8192
    w, sw = random_bytes(0, 256, E, N, K // 2), random_bytes(120, 130, E, N, K // 32)
    a, sa = matrix(R, K, 1)
    got = impl("moe_mxfp4_grouped_gemm").run(a, sa, w, sw, torch.tensor([0] * E + [R], dtype=torch.int32, device="cuda"))
    cols = torch.tensor([0, 33, N // 2 + 1, *range(N - 300, N)], device="cuda")
    x, v = dequant_ref.values(a, sa), dequant_ref.values(w[E - 1][cols], sw[E - 1][cols])
    check_close(got[:, cols], x @ v.t(), x.abs() @ v.abs().t(), K)


def test_results_behind_4_gib(gpu):
    say("gemm far results")
    M, N, K = 70000, 40000, 32
    a, sa, w, sw = *matrix(M, K, 1), *matrix(N, K, 2)
    got = impl("mxfp4_gemm").run(a, sa, w, sw)
    for rows in (slice(0, 40), slice(M // 2, M // 2 + 40), slice(M - 300, M)):
        x, v = dequant_ref.values(a[rows], sa[rows]), dequant_ref.values(w, sw)
        check_close(got[rows], x @ v.t(), x.abs() @ v.abs().t(), K)


@pytest.mark.parametrize("gated", [False, True])
def test_quantisation_behind_4_gib(gpu, gated):
    say("quant far rows", gated)
    M, K = 65539, 32800
    x = torch.randn(300, K, dtype=torch.bfloat16, device="cuda").repeat(-(-M // 300), 1)[:M]
    codes, scales = impl("mxfp4_quant").run(x, gated=gated) if not gated else impl("mxfp4_quant").run(x[:, :32768], gated=True)
    rows = torch.tensor([0, M // 2, M - 2, M - 1], device="cuda")
    want = quant_ref.run((x[rows, :32768] if gated else x[rows]).cpu(), gated)
    assert torch.equal(codes[rows].cpu(), want[0]) and torch.equal(scales[rows].cpu(), want[1])
    if not gated:
        back = impl("mxfp4_dequant").run(codes, scales)
        assert torch.equal(back[rows].double(), dequant_ref.values(codes[rows], scales[rows]).bfloat16().double())


# ----------------------------------------------------------------------------- routing


def check_route(logits, k, bias=None, scale=1.0, renormalize=True, **kw):
    w, ids = impl("moe_expert_routing").run(logits.cuda(), k, None if bias is None else bias.cuda(), scale=scale,
                                            renormalize=renormalize, **kw)
    want = route_ref.run(logits, k, bias, scale=scale, renormalize=renormalize, **kw)
    assert torch.equal(ids.cpu(), want[1])
    # both rounded once to fp32 from 64 bits
    torch.testing.assert_close(w.cpu(), want[0], rtol=2.0 ** -23, atol=2.0 ** -149, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T_,E,k,groups,top_groups,group_top", [
    (1, 256, 8, 8, 4, 2), (67, 256, 8, 8, 4, 2), (130, 60, 4, 1, 1, 1), (33, 384, 7, 16, 11, 1), (20, 1024, 32, 64, 3, 2),
    (9, 1, 1, 1, 1, 1), (11, 7, 7, 1, 1, 1), (50, 64, 6, 4, 1, 2), (40, 160, 6, 8, 3, 1), (21, 500, 3, 5, 2, 2),
    (70, 128, 2, 2, 2, 2), (300, 8, 2, 1, 1, 1), (19, 1024, 8, 8, 4, 2), (23, 512, 8, 1, 1, 1), (10, 768, 8, 16, 5, 2),
    (13, 700, 5, 7, 3, 1), (37, 12, 3, 2, 1, 2), (31, 90, 8, 5, 2, 2), (31, 90, 5, 3, 2, 1), (15, 90, 8, 15, 7, 2),
    (9, 128, 8, 64, 9, 2), (258, 250, 8, 1, 1, 1)])
def test_routing(gpu, T_, E, k, groups, top_groups, group_top, score, dtype):
    say("routing", T_, E, k, groups, score, dtype)
    g = gen(E + k)
    logits = (torch.randn(T_, E, generator=g) * 2).to(dtype)
    bias = torch.randn(E, generator=g) * 0.1
    kw = dict(groups=groups, top_groups=top_groups, group_top=group_top, score=score)
    check_route(logits, k, bias, 2.5, **kw)
    check_route(logits, k, None, 1.0, False, **kw)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups", [(16, 4), (256, 8), (256, 1), (60, 1), (96, 8)])
def test_routing_of_ties_masks_and_nan(gpu, E, groups, score):
    say("routing ties", E, groups, score)
    inf, g = float("inf"), gen(E)
    logits = torch.randint(-2, 3, (64, E), generator=g).float()       # many equal choices
    logits[0] = 0
    logits[1] = -inf
    logits[2] = -inf
    logits[2, E - 1] = 1.0
    logits[3, E // 2] = float("nan")
    logits[4, :] = float("nan")
    logits[5] = 800.0
    logits[6] = -800.0
    logits[7] = 50.0 + torch.arange(E)                                 # sigmoids that round to 1
    logits[8] = -60.0 - torch.arange(E) / 8
    logits[9, 3] = inf
    logits[10, ::2] = -inf
    logits[11] = -0.0
    kw = dict(groups=groups, top_groups=max(1, groups // 2), group_top=2, score=score)
    for k in (1, 4, 6):
        check_route(logits, k, None, **kw)
        check_route(logits, k, torch.randint(-1, 2, (E,), generator=g).float(), **kw)
        check_route(logits.half(), k, torch.zeros(E), **kw)
    bias = torch.zeros(E)
    bias[:E // 2], bias[E - 1] = -inf, -0.0
    check_route(logits, 4, bias, renormalize=False, **kw)


def test_routing_next_to_borders(gpu):
    """Scores that fp32 cannot tell apart: choices one fp64 step above or below their neighbours'."""
    say("routing borders")
    g = gen(1)
    logits = torch.randn(200, 64, generator=g)
    other = torch.nextafter(logits, torch.full_like(logits, 9.0))
    check_route(torch.cat((logits, other), dim=1)[:, torch.randperm(128, generator=g)], 8, score="softmax")
    check_route(torch.cat((logits, other), dim=1)[:, torch.randperm(128, generator=g)], 8, torch.rand(128, generator=g) * 1e-7,
                groups=4, top_groups=2, group_top=2, score="sigmoid")


def test_routing_takes_any_strides(gpu):
    say("routing strides")
    x = torch.randn(40, 3, 64, generator=gen(2))
    for layout in (lambda x: x[:, 1], lambda x: x[:, 0, 5:45], lambda x: x[:, 2].t().contiguous().t(),
                   lambda x: x[:1, 0].expand(6, 64), lambda x: x[:0, 0], lambda x: x[0].t()[:, :1].expand(64, 5)):
        w, ids = impl("moe_expert_routing").run(layout(x.cuda()), 3, score="sigmoid")
        want = route_ref.run(layout(x), 3, score="sigmoid")
        assert torch.equal(ids.cpu(), want[1]) and w.shape == want[0].shape


def test_routing_behind_4_gib(gpu):
    say("routing far rows")
    rows = (torch.randn(1000, 1024, generator=gen(3)) * 2).bfloat16()
    logits = rows.cuda().repeat(2200, 1)
    want = route_ref.run(rows[-50:], 8)
    for k in (8, 9):                                       # lanes, rows
        w, ids = impl("moe_expert_routing").run(logits, k)
        assert torch.equal(ids[-50:, :8].cpu(), want[1]) and torch.equal(ids[-1000:], ids[:1000]) and torch.equal(w[-1000:], w[:1000])


@pytest.mark.parametrize("E,k,groups,kernel", [
    (60, 4, 1, "route_lanes"), (256, 8, 8, "route_lanes"), (256, 9, 8, "route_rows"), (90, 8, 9, "route_rows")])
def test_routing_says_which_kernel_ran(gpu, E, k, groups, kernel):
    say("routing config", E, k, groups)
    check_route(torch.randn(5, E, generator=gen(1)), k, groups=groups, top_groups=groups)
    assert impl("moe_expert_routing").get_last_config()["kernel"] == kernel


# ----------------------------------------------------------------------------- together


def layer(x, logits, bias, w13, w2, E, k):
    """An expert layer: routing, tokens quantised once, gate and up, silu(gate) * up quantised, down, weighted sum."""
    weights, ids = impl("moe_expert_routing").run(logits, k, bias, groups=4, top_groups=2, group_top=2, score="sigmoid",
                                                  scale=2.5)
    pairs, offsets = experts.align(ids, E)
    h = impl("moe_mxfp4_grouped_gemm").run(*impl("mxfp4_quant").run(x), *w13, offsets, gather=pairs, topk=k, dtype=x.dtype)
    act = impl("mxfp4_quant").run(h, gated=True)
    y = impl("moe_mxfp4_grouped_gemm").run(*act, *w2, offsets, scatter=pairs, weights=weights.flatten(), dtype=x.dtype)
    return experts.combine(y, ids, E), (weights, ids, pairs, offsets, h, act, y)


def make_layer(tokens, E, H, I, dtype, seed):
    g = gen(seed)
    x = torch.randn(tokens, H, generator=g).to(dtype).cuda()
    logits, bias = torch.randn(tokens, E, generator=g).cuda(), (torch.randn(E, generator=g) * 0.1).cuda()
    w13, w2 = ([t.cuda() for t in mxfp4_matrix(torch.randn(E, n, m, generator=g) * m ** -0.5, "cpu")]
               for n, m in ((2 * I, H), (H, I)))
    return x, logits, bias, w13, w2


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tokens", [1, 19, 300])
def test_an_expert_layer(gpu, tokens, dtype):
    say("layer", tokens, dtype)
    E, k, H, I = 16, 4, 512, 352
    x, logits, bias, w13, w2 = make_layer(tokens, E, H, I, dtype, tokens)
    out, (weights, ids, pairs, offsets, h, act, y) = layer(x, logits, bias, w13, w2, E, k)
    # step by step, each from what the step before gave
    want = route_ref.run(logits.cpu(), k, bias.cpu(), 4, 2, 2, "sigmoid", scale=2.5)
    assert torch.equal(ids.cpu(), want[1])
    flat = ids.flatten().long()
    assert torch.equal(pairs.long(), torch.sort(flat, stable=True).indices)
    assert torch.equal(offsets[1:].long(), torch.bincount(flat, minlength=E).cumsum(0))
    check_grouped(*impl("mxfp4_quant").run(x), *w13, offsets, dtype, H, gather=pairs, topk=k)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(act, quant_ref.run(h.cpu(), True)))
    check_grouped(*act, *w2, offsets, dtype, I, scatter=pairs, weights=weights.flatten())
    total = y.view(tokens, k, H).double()
    t = torch.finfo(dtype)  # k - 1 fp32 additions, one rounding
    bound = t.eps / 2 * total.sum(dim=1).abs() + k * 2.0 ** -23 * total.abs().sum(dim=1) + t.smallest_normal * t.eps
    assert bool(((out.double() - total.sum(dim=1)).abs() <= bound).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tokens,k,H", [(1, 1, 8), (33, 8, 264), (70, 12, 1032), (5, 32, 16)])
def test_combine(gpu, tokens, k, H, dtype):
    """Additions in fp32 in slot order and one rounding: one right answer."""
    say("combine", tokens, k, H, dtype)
    g = gen(k)
    y = (torch.randn(tokens * k, H, generator=g) * torch.exp2(torch.randint(-9, 10, (tokens * k, 1), generator=g).float())).to(dtype)
    y[0, :6] = torch.tensor([float("inf"), float("-inf"), float("nan"), torch.finfo(dtype).max, -0.0, torch.finfo(dtype).tiny / 4])
    ids = torch.randint(-1, 9, (tokens, k), generator=g).int()
    ids[0, 0] = 0
    total = torch.zeros(tokens, H)
    for j in range(k):
        row = y.view(tokens, k, H)[:, j].float()
        total = torch.where(((ids[:, j] >= 0) & (ids[:, j] < 8))[:, None], total + row, total)
    torch.testing.assert_close(experts.combine(y.cuda(), ids.cuda(), 8).cpu(), total.to(dtype), rtol=0, atol=0, equal_nan=True)


def test_padded_tokens_are_routed_nowhere(gpu):
    say("layer padding")
    E, k, H = 16, 4, 256
    x, logits, bias, w13, w2 = make_layer(20, E, H, 64, torch.bfloat16, 5)
    weights, ids = impl("moe_expert_routing").run(logits, k, bias)
    ids[7:] = -1
    pairs, offsets = experts.align(ids, E)
    assert int(offsets[E]) == 7 * k
    pairs[7 * k:] = 2 ** 31 - 1
    y = torch.full((20 * k, H), float("nan"), dtype=torch.bfloat16, device="cuda")
    act = impl("mxfp4_quant").run(torch.randn(20 * k, 64, generator=gen(3)).cuda())
    impl("moe_mxfp4_grouped_gemm").run(*act, *w2, offsets, scatter=pairs, weights=weights.flatten(), out=y)
    assert bool(torch.isnan(y[7 * k:]).all()) and bool(torch.isfinite(y[:7 * k]).all())
    out = experts.combine(y, ids, E)
    assert bool(torch.isfinite(out[:7]).all()) and not bool(out[7:].any())


def test_a_captured_layer_replays(gpu):
    say("layer graph")
    E, k = 16, 4
    x, logits, bias, w13, w2 = make_layer(33, E, 512, 160, torch.bfloat16, 6)
    want = layer(x, logits, bias, w13, w2, E, k)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer(x, logits, bias, w13, w2, E, k)
    for i in range(4):
        say("replay", i)
        if i == 2:
            fresh = make_layer(33, E, 512, 160, torch.bfloat16, 7)
            for a, b in zip((x, logits), fresh):
                a.copy_(b)
            want = layer(x, logits, bias, w13, w2, E, k)[0]
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(layer(x, logits, bias, w13, w2, E, k)[0], want)


def test_layers_on_two_streams(gpu):
    say("layer streams")
    E, k = 16, 4
    inputs = [make_layer(40, E, 512, 160, torch.float16, s) for s in (1, 2)]
    want = [layer(*i, E, k)[0] for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for i, s in zip(inputs, streams):
            with torch.cuda.stream(s):
                got.append(layer(*i, E, k)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[n % 2]) for n, g in enumerate(got))


def test_tensors_off_the_gpu_are_refused(gpu):
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="cpu"):
        impl("mxfp4_quant").run(x)
    with pytest.raises(ValueError, match="cpu"):
        impl("moe_expert_routing").run(x, 2)
    a, sa = matrix(4, 64, 1)
    with pytest.raises(ValueError, match="cpu"):
        impl("mxfp4_gemm").run(a, sa, a.cpu(), sa)


# ----------------------------------------------------------------------------- the harness


CASES = [
    ("moe_expert_routing", dict(T=100, E=256), torch.float32),
    ("moe_expert_routing", dict(T=100, E=64, groups=1, top_groups=1, score="softmax"), torch.bfloat16),
    ("mxfp4_quant", dict(M=100, K=1408), torch.float16),
    ("mxfp4_quant", dict(M=100, K=1408, gated=True), torch.bfloat16),
    ("mxfp4_dequant", dict(M=100, K=2912), torch.bfloat16),
    ("mxfp4_gemm", dict(M=20, N=200, K=1408), torch.bfloat16),
    ("mxfp4_gemm", dict(M=300, N=264, K=736), torch.float16),
]


def test_every_expert_operator_has_a_case():
    from tilebench_amd.paths import list_expert_operators

    # the grouped product's rows depend on its routing: the checks below need inputs of one shape
    assert {op for op, *_ in CASES} | {"moe_mxfp4_grouped_gemm"} == set(list_expert_operators())


@pytest.mark.parametrize("op,case,dtype", CASES, ids=[f"{op}-{i}" for i, (op, *_) in enumerate(CASES)])
def test_fresh_inputs_same_address_and_repeat(gpu, op, case, dtype):
    import importlib
    import itertools

    import yaml

    from tilebench_amd.core.anticache import CHECKS, numerical_checks
    from tilebench_amd.core.verifier import config_per_output, config_tolerance
    from tilebench_amd.paths import operator_config

    say("anticache", op, case, dtype)
    cfg = yaml.safe_load(open(operator_config(op)))["verify"]
    atol, rtol = config_tolerance(cfg, None)
    seeds = itertools.count(50)

    def make():
        x = T.get_generator(op)(**case, dtype=dtype, seed=next(seeds), device="cpu")
        return tuple(t.to("cuda") if isinstance(t, torch.Tensor) else t for t in x)

    reference = importlib.import_module(f"tilebench_amd.benchmarks.experts.{op}.impl_torch").run
    res = numerical_checks(impl(op).run, reference, make, atol=atol, rtol=rtol, per_output=config_per_output(cfg, None))
    assert [r.name for r in res] == list(CHECKS), res[-1].message
    assert all(r.ok for r in res), [r.message for r in res if not r.ok]
    assert not any(r.aliased_inputs or r.mutated_inputs for r in res)


@pytest.mark.parametrize("op,case", [
    ("moe_expert_routing", dict(T=64)), ("mxfp4_quant", dict(M=64, K=512)), ("mxfp4_dequant", dict(M=64, K=512)),
    ("mxfp4_gemm", dict(M=64, N=128, K=512)), ("moe_mxfp4_grouped_gemm", dict(tokens=16, experts=8, K=512, N=96))])
def test_the_engine_runs_it(gpu, op, case):
    from tilebench_amd.core import engine

    say("engine", op)
    rows = engine.run_benchmark_suite(op, benchmark_overrides={"case_indices": [0, 1], "case_overrides": case},
                                      enabled_backends=["hip"])
    assert rows and all(r["hip_ok"] for r in rows), [r["hip_err"] for r in rows]
    assert all(r["hip_config"] for r in rows)
