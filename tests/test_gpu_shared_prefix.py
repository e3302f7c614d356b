"""Paged attention over shared prefixes on the GPU against the formula in fp64 on
the CPU (bounds: shared_prefix_cases.check)."""
import pytest
import torch

from tests.shared_prefix_cases import check, check_far_scales, far_scales, make, reference
from tilebench_amd.data import tensors as T

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _say(*a):
    print("[gpu case]", *a, flush=True)


def _to(x, gpu):
    return [v.to(gpu) if isinstance(v, torch.Tensor) else v for v in x]


def _run(x, gpu):
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    out = impl_hip.run(*_to(x, gpu))
    torch.cuda.synchronize()
    assert out[0].dtype == x[0].dtype and out[0].shape == x[0].shape and out[1].dtype == torch.float32
    return out


ONES = [1] * 40
CASES = {
    # decode without prefixes: lengths around steps of 32 and 64 tokens and pages
    "decode": dict(n_q=[1] * 9, lens=[1, 2, 15, 16, 17, 31, 33, 64, 65]),
    "decode_long": dict(n_q=[1, 1], lens=[3001, 257], D=128),
    "one_token": dict(n_q=[1], lens=[1], Hq=1, Hkv=1),
    "empty_sequences": dict(n_q=[1, 0, 1, 0, 0], lens=[0, 7, 40, 0, 3], pad=3, spare=2),
    "many_sequences": dict(n_q=[1] * 300, lens=[(7 * i) % 90 for i in range(300)], Hq=2, Hkv=2),
    # few rows: groups of up to 32 rows
    "rows_16": dict(n_q=[4, 4], lens=[50, 4], prefix=[100], page=32),
    "rows_32": dict(n_q=[2, 2, 4], lens=[50, 2, 90], prefix=[300], D=128, page=64),
    "rows_16_long": dict(n_q=[2, 2], lens=[50, 4], prefix=[1500], page=32, pad=1),
    "rows_12_groups": dict(n_q=[1, 1, 1, 2, 1], lens=[50, 4, 0, 300, 7], prefix=[1500, 0, 900], bounds=[0, 2, 3, 5],
                           D=128, page=32),
    "joint_groups": dict(n_q=[1, 1, 1, 2, 1, 0], lens=[50, 4, 0, 300, 7, 2], prefix=[150, 0, 500], bounds=[0, 2, 3, 6],
                         page=32, pad=2),
    "many_groups": dict(n_q=[1] * 150, lens=[(5 * i) % 40 for i in range(150)], prefix=[(17 * i) % 300 for i in range(75)],
                        bounds=[2 * i for i in range(76)], Hq=20, Hkv=2, page=8),
    "many_in_a_group": dict(n_q=[1] * 150, lens=[(5 * i) % 40 for i in range(150)], prefix=[1100], page=16),
    "many_mixed": dict(n_q=[1 + 7 * (i % 5 == 0) for i in range(150)], lens=[9 + (5 * i) % 40 for i in range(150)],
                       prefix=[100], page=16),
    "mqa_20_rows": dict(n_q=[1, 1], lens=[30, 200], prefix=[500], Hq=20, Hkv=1, D=128),
    # row tiles
    "tile_ragged": dict(n_q=ONES, lens=[(11 * i) % 70 + 1 for i in range(40)], prefix=[1000], page=32),
    "tile_d128": dict(n_q=ONES, lens=[(13 * i) % 200 + 1 for i in range(40)], prefix=[777], D=128, page=64),
    "tile_one_token_prefix": dict(n_q=ONES, lens=[5] * 40, prefix=[1]),
    "tile_no_prefix_length": dict(n_q=ONES, lens=[5] * 40, prefix=[0]),
    "groups": dict(n_q=[1, 2, 1, 9, 1, 1, 0, 30, 1, 1], lens=[5, 6, 70, 40, 1, 0, 9, 31, 2, 3],
                   prefix=[130, 0, 64, 1000], bounds=[0, 3, 4, 4, 10], page=8),
    "mixed": dict(n_q=[1, 90, 1, 1, 33, 2], lens=[60, 100, 1, 9, 33, 64], prefix=[200], D=128, page=16),
    "mixed_no_prefix": dict(n_q=[1, 90, 1, 1, 33, 2], lens=[60, 100, 1, 9, 33, 64], page=16, pad=5),
    "chunks": dict(n_q=[130, 257, 64], lens=[130, 300, 1000], prefix=[65], page=64, D=128),
    "chunk_long": dict(n_q=[200], lens=[4000], Hq=4, Hkv=1, D=128, page=128),
    "queries_before_tokens": dict(n_q=[50, 3], lens=[20, 1], prefix=[10], page=4),
    "queries_before_all": dict(n_q=[50, 40], lens=[0, 0], prefix=[0]),
    "mha": dict(n_q=[1, 70, 1], lens=[100, 90, 3], prefix=[99], Hq=5, Hkv=5),
    "mqa": dict(n_q=[1, 3, 1], lens=[100, 90, 3], prefix=[99], Hq=71, Hkv=1, page=1),
    "group_of_five": dict(n_q=[1, 30, 7, 6], lens=[100, 90, 30, 30], prefix=[300], Hq=10, Hkv=2, D=128),
    "page_1": dict(n_q=[1, 30], lens=[100, 90], prefix=[150], page=1),
    "page_4096": dict(n_q=[1, 30], lens=[100, 4500], prefix=[150], page=4096),
    "peaked": dict(n_q=[1, 40], lens=[900, 900], prefix=[500], q_scale=30.0),
}


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("name", CASES)
def test_attention_matches_the_formula(gpu, name, dtype, cache):
    _say("attention", name, dtype, cache)
    x = make(**CASES[name], dtype=dtype, cache=cache, seed=len(name))
    check(_run(x, gpu), x)


# Calls whose partial results would take more than 512 MiB with slots for every row: only rows that need some have them.
COMPACT = {
    # rounds of whole tiles and a split last one; sequences of up to 16 rows among longer ones
    "prompts": dict(n_q=[200] * 36 + [1, 2, 0, 1, 17, 3], lens=[200 + i for i in range(36)] + [50, 2, 9, 300, 40, 3],
                    prefix=[300], Hq=64, Hkv=8, pad=3),
    "prompts_groups": dict(n_q=[200] * 36 + [1, 2, 0, 1, 17, 3], lens=[200 + i for i in range(36)] + [50, 2, 9, 300, 40, 3],
                           prefix=[300, 0, 120], bounds=[0, 10, 25, 42], Hq=64, Hkv=8, pad=3),
    "prompts_alone": dict(n_q=[1, 2, 0, 1, 17, 3] + [200] * 36, lens=[50, 2, 9, 300, 40, 3] + [200 + i for i in range(36)],
                          Hq=64, Hkv=8, pad=3),
    "mixed": dict(n_q=[3 + 30 * (i % 40 == 0) for i in range(1430)], lens=[40 + i % 200 for i in range(1430)], prefix=[700],
                  Hq=64, Hkv=8),
    "decodes": dict(n_q=[1] * 1200, lens=[1 + i % 90 for i in range(1200)], prefix=[2100], Hq=64, Hkv=8, spare=400),
    # fewer tiles, shared out by their steps: some are split and some are not
    "tenants": dict(n_q=[2] * 150, lens=[2 + i % 90 for i in range(150)],
                    prefix=[(17 * i) % 300 + 3000 * (i % 50 == 7) for i in range(150)], bounds=list(range(151)), Hq=32,
                    Hkv=8, D=128, spare=1024),
    "tenants_drafts": dict(n_q=[1 + 10 * (i % 2) for i in range(150)], lens=[11 + i % 90 for i in range(150)],
                           prefix=[(17 * i) % 300 + 3000 * (i % 50 == 7) for i in range(150)], bounds=list(range(151)),
                           Hq=32, Hkv=8, D=128, spare=1024),
    "five_tenants": dict(n_q=[1] * 300, lens=[1 + i % 90 for i in range(300)], prefix=[900, 0, 3000, 20, 700],
                         bounds=[0, 60, 100, 180, 181, 300], Hq=32, Hkv=8, D=128, spare=1024),
    "one_tenant": dict(n_q=[1] * 500, lens=[1 + i % 90 for i in range(500)], prefix=[900], Hq=32, Hkv=8, D=128, spare=246),
}


@pytest.mark.parametrize("name,dtype,cache", [(name, F16, "same") for name in COMPACT] +
                         [(name, BF16, "e4m3") for name in ("prompts", "tenants_drafts")])
def test_slots_only_for_rows_that_need_them(gpu, name, dtype, cache):
    _say("attention compact", name, dtype, cache)
    kw = dict(COMPACT[name], dtype=dtype, cache=cache, seed=len(name))
    x = make(**kw)
    got = _run(x, gpu)
    check(got, make(**dict(kw, spare=0)))  # the same call with tables as wide as they need to be
    again = _run(x, gpu)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("name", ["prompts", "five_tenants"])
def test_replays_with_slots_only_where_needed(gpu, name):
    """Two captured calls, replayed in turn with other contents, eager calls between them."""
    _say("attention compact graphs", name)
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    xs = [_to(make(**COMPACT[name], seed=80 + i), gpu) for i in range(2)]
    impl_hip.run(*xs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(impl_hip.run(*x))
    for seed in range(3):
        new = [_to(make(**COMPACT[name], seed=90 + 2 * seed + i), gpu) for i in range(2)]
        for x, y in zip(xs, new):
            y[7] = torch.clamp(y[7] - seed, min=0)     # other lengths, the same tables
            for a, b in zip(x, y):
                if isinstance(a, torch.Tensor):
                    a.copy_(b)
        want = [impl_hip.run(*y) for y in new]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_splits_of_long_prefixes_and_scales(gpu):
    for seed, (scale, kw) in enumerate([
            (None, dict(n_q=[1] * 3, lens=[9, 700, 33], prefix=[20000], Hq=16, Hkv=2, D=128, page=64)),
            (0.5, dict(n_q=[1] * 50, lens=[9] * 50, prefix=[9000], Hq=8, Hkv=2, D=64, page=64, dtype=BF16)),
            (0.0, dict(n_q=[2] * 9, lens=[9] * 9, prefix=[300], Hq=8, Hkv=2, D=64)),
            (-0.125, dict(n_q=[2] * 9, lens=[9] * 9, prefix=[300], Hq=8, Hkv=2, D=64))]):
        _say("attention splits", scale, kw)
        x = make(**kw, seed=seed)
        x[10] = scale
        got = _run(x, gpu)
        if scale == 0.0:
            x[10] = 0.0
            want, lse, mean = reference(x)
            # all weights are equal: the scores are exact
            x[10] = 1e-30
            check(got, x, (want, lse, mean))
        elif scale is not None and scale < 0:
            ref = reference(x)
            x[10] = -scale
            check(got, x, ref)
        else:
            check(got, x)


# value scales from those of values around 1e-4 to those of values around 1e4, alone and mixed within a sequence
@pytest.mark.parametrize("low, high", [(-14, -14), (-7, -7), (12, 12), (-14, 12)])
@pytest.mark.parametrize("kw", [
    dict(n_q=[1, 2], lens=[200, 70], prefix=[500]), dict(n_q=[1, 2], lens=[900, 70], prefix=[1100], D=128),
    dict(n_q=ONES, lens=[300] * 40, prefix=[900], D=128), dict(n_q=[90, 3], lens=[800, 20], prefix=[30])],
    ids=["joint", "few", "tile", "chunk"])
def test_value_scales_of_any_size(gpu, kw, low, high):
    for dtype in (F16, BF16):
        _say("value scales", kw, low, high, dtype)
        x = make(**kw, cache="e4m3", dtype=dtype, seed=low + 20)
        g = torch.Generator().manual_seed(high)
        x[12] *= 2.0 ** torch.randint(low, high + 1, x[12].shape, generator=g)
        check(_run(x, gpu), x)


@pytest.mark.parametrize("ratio", [2.0 ** 30, 2.0 ** 50, 2.0 ** -50, 0.0])
@pytest.mark.parametrize("kw", [
    dict(n_q=[1, 2], lens=[200, 70], prefix=[500]), dict(n_q=[1, 2], lens=[900, 70], prefix=[1100], D=128),
    dict(n_q=ONES, lens=[300] * 40, prefix=[900], D=128), dict(n_q=[90, 3], lens=[800, 20], prefix=[30])],
    ids=["joint", "few", "tile", "chunk"])
def test_values_beside_others_of_no_weight(gpu, kw, ratio):
    """Tokens of next to no weight whose values are far larger or smaller than those that count, or zero."""
    for dtype in (F16, BF16):
        _say("far scales", kw, ratio, dtype)
        x = make(**kw, cache="e4m3", dtype=dtype, seed=31)
        far_scales(x, ratio)
        check_far_scales(_run(x, gpu), x)


@pytest.mark.parametrize("kw", [
    dict(n_q=[1, 1], lens=[20, 70], prefix=[40]), dict(n_q=[1, 2], lens=[20, 70], prefix=[1100]), dict(n_q=ONES, lens=[20] * 40, prefix=[90], D=128),
    dict(n_q=[70, 3], lens=[80, 20], prefix=[30], D=128), dict(n_q=[4, 2, 1], lens=[40, 3, 9])],
    ids=["joint", "few", "tile", "chunk", "drafts"])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_values_outside_a_row_s_tokens_leave_no_trace(gpu, kw, cache):
    """NaN and infinities in unused slots and pages; in tokens after a query's own;
    in keys and values that a row does see (there the result is NaN or that infinity)."""
    _say("attention special values", kw, cache)
    x = make(**kw, cache=cache, seed=5, spare=1)
    P = x[1].shape[2]
    clean = _run(x, gpu)
    # slots behind the last token of every sequence and prefix
    y = [v.clone() if isinstance(v, torch.Tensor) else v for v in x]
    nan = torch.tensor(float("nan"))
    for table, lens in ((y[6], y[7]), (y[3], y[4])):
        if table is None:
            continue
        for row, n in zip(table, lens.tolist()):
            if n % P:
                page = int(row[n // P])
                for c in y[1:3]:
                    c[page, :, n % P:] = nan.to(c.dtype)
                for s in y[11:]:
                    s[page, :, n % P:] = float("nan")
    got = _run(y, gpu)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # the last own token of every sequence: only its last query sees it
    for which, value in ((2, float("nan")), (2, float("inf")), (2, float("-inf")), (1, float("nan"))):
        if cache == "e4m3" and value == value:
            continue  # e4m3 has no infinities
        z = [v.clone() if isinstance(v, torch.Tensor) else v for v in x]
        for row, n in zip(z[6], z[7].tolist()):
            z[which][int(row[(n - 1) // P]), 0, (n - 1) % P, 3] = torch.tensor(value).to(z[which].dtype)
        check(_run(z, gpu), z, reference(z))


def test_malformed_lengths_and_ids_stay_inside(gpu):
    """Lengths past the tables, negative ones, ids outside the pool: clamped, as in the reference."""
    _say("attention malformed")
    x = make([1, 2, 40], [30, 9, 60], prefix=[33, 20], bounds=[0, 1, 3], seed=7)
    x[7][0], x[7][1], x[4][0], x[4][1] = 10 ** 6, -5, 2 ** 31 - 1, -1
    x[6][2, 1], x[6][0, 0], x[3][0, 1] = -3, 10 ** 9, 2 ** 31 - 1
    check(_run(x, gpu), x)
    # cu_q and group_offsets out of order: in bounds and finite
    y = make([1, 2, 40], [30, 9, 60], prefix=[33, 20], bounds=[0, 1, 3], seed=7)
    for bad in ([0, 50, 10, 43], [5, 1, 100, 2], [-9, 1, 3, 10 ** 9]):
        y[8] = torch.tensor(bad, dtype=torch.int32)
        out, _ = _run(y, gpu)
        assert out.shape == y[0].shape
    y[8], y[5] = x[8], torch.tensor([7, -2, 99], dtype=torch.int32)
    _run(y, gpu)


@pytest.mark.parametrize("kw", [
    dict(n_q=[1, 2, 40], lens=[30, 9, 60], prefix=[33, 20], bounds=[0, 1, 3]),                           # tiles
    dict(n_q=[1, 2, 1, 1], lens=[30, 9, 60, 4], prefix=[33, 20], bounds=[0, 1, 4]),                      # a block each
    dict(n_q=[1, 2, 1, 1], lens=[30, 9, 900, 4], prefix=[1500, 20], bounds=[0, 1, 4], D=128),            # streams
    dict(n_q=[1, 1, 1, 1] * 40, lens=[30, 9, 60, 4] * 40, prefix=[1100] * 80, bounds=[2 * i for i in range(81)]),
    COMPACT["tenants_drafts"]], ids=["tiles", "each", "streams", "groups", "compact"])
def test_offsets_out_of_order_leave_other_memory_alone(gpu, kw):
    """cu_q and group_offsets that do not ascend: their rows hold anything, but nothing around the buffers changes."""
    import ctypes

    from tilebench_amd import runtime as rt

    _say("attention offsets out of order", len(kw["n_q"]))
    x = make(**kw, seed=7)
    y = _to(x, gpu)
    T, Hq, D = x[0].shape
    (pages, Hkv, page, _), (G, Wp), (B, W) = x[1].shape, x[3].shape, x[6].shape
    need = ctypes.c_int64(0)
    rt.call("tb_shared_prefix_attention_workspace_size", T, Hq, Hkv, D, G, Wp, B, W, page, x[9], 1, ctypes.byref(need))
    guard = 1 << 16
    buffers = [torch.full((n + 2 * guard,), 0xA5, dtype=torch.uint8, device=gpu)
               for n in (T * Hq * D * 2, T * Hq * 4, need.value)]
    g = torch.Generator().manual_seed(1)
    backwards = lambda t: t.flip(0).contiguous()                                     # noqa: E731
    wild = lambda t: torch.randint(-9, T + 90, t.shape, generator=g).int()           # noqa: E731
    for cu, go in ((backwards(x[8]), x[5]), (x[8], backwards(x[5])), (wild(x[8]), x[5]), (x[8], wild(x[5])),
                   (wild(x[8]), wild(x[5])), (x[8], torch.full_like(x[5], 0)),
                   (x[8], torch.tensor([0, B] * len(x[5])).int()[:len(x[5])])):
        cu, go = cu.to(gpu), go.to(gpu)
        out, lse, ws = (b.data_ptr() + guard for b in buffers)
        rt.call("tb_shared_prefix_attention", y[0].data_ptr(), y[1].data_ptr(), y[2].data_ptr(), None, None,
                y[3].data_ptr(), y[4].data_ptr(), go.data_ptr(), y[6].data_ptr(), y[7].data_ptr(), cu.data_ptr(), out,
                lse, T, Hq, Hkv, D, G, Wp, B, W, x[9], pages, page, Hq * D, D, Hkv * page * D, page * D, D, 0, 0, 0,
                D ** -0.5, 1, 1, ws if need.value else None, need.value, rt.stream_handle(y[0].get_device()))
        torch.cuda.synchronize()
        for b in buffers:
            assert bool((b[:guard] == 0xA5).all()) and bool((b[-guard:] == 0xA5).all())


def test_more_queries_than_announced_are_empty_or_right(gpu):
    _say("attention max_q too small")
    x = make([60, 1], [60, 9], Hq=4, Hkv=2, seed=8)
    x[9] = 1
    out, lse = _run(x, gpu)
    assert bool((out[:60] == 0).all()) and bool((lse[:60] == -float("inf")).all())
    x[9] = 60
    ref = reference(x)
    assert float((out[60].cpu().double() - ref[0][60]).abs().max()) < 1e-2


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_layouts_give_the_same_bits(gpu, cache):
    """q from a fused projection, [pages, page, heads, D] pools, pools with keys beside values."""
    _say("attention layouts", cache)
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    x = _to(make([1, 50, 2], [70, 60, 9], prefix=[100], D=64, cache=cache, seed=9), gpu)
    want = impl_hip.run(*x)
    u8 = lambda c: c.view(torch.uint8) if c.element_size() == 1 else c  # noqa: E731
    wide = torch.zeros(x[0].shape[0], 3 * 8 * 64 + 8, dtype=F16, device=gpu)
    q = wide[:, 8:8 + 8 * 64].view(-1, 8, 64)
    q.copy_(x[0])
    odd = wide[:, 3:3 + 8 * 64].view(-1, 8, 64)  # not 16-byte aligned: copied
    nhd = [u8(c).transpose(1, 2).contiguous().transpose(1, 2).view(c.dtype) for c in x[1:3]]
    both = torch.stack([u8(c) for c in x[1:3]], dim=1).contiguous()
    side = [both[:, i].view(x[1].dtype) for i in range(2)]
    for pools in (nhd, side):
        got = impl_hip.run(q, *pools, *x[3:])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd.copy_(x[0])
    got = impl_hip.run(odd, *x[1:])
    assert torch.equal(got[0], want[0])
    again = impl_hip.run(*x)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("T,Hq,Hkv", [(1, 8, 2), (1, 1, 1), (3, 1, 1)])
def test_one_token_of_an_odd_projection(gpu, T, Hq, Hkv):
    """Dimensions of size 1 keep odd strides in PyTorch's copies."""
    _say("attention odd strides", T, Hq, Hkv)
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    x = _to(make([1] * T, [9] * T, prefix=[30], Hq=Hq, Hkv=Hkv, seed=12), gpu)
    want = impl_hip.run(*x)
    for shift, gap in ((0, 3), (3, 0), (3, 5)):
        wide = torch.zeros(T + 1, Hq * 64 + shift + gap, dtype=F16, device=gpu)
        q = wide[:, shift:shift + Hq * 64].view(T + 1, Hq, 64)[1:]
        q.copy_(x[0])
        got = impl_hip.run(q, *x[1:])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_past_4_gib_of_cache(gpu):
    """Pages at the end of a 6 GiB pool."""
    _say("attention 64-bit offsets")
    x = make([1, 40], [70, 60], prefix=[100], Hq=16, Hkv=8, D=128, page=64, seed=10)
    n = x[1].shape[0]
    pages = 6 * 2 ** 30 // (8 * 64 * 128 * 2)
    y = _to(x, gpu)
    for i in (1, 2):
        pool = torch.zeros(pages, 8, 64, 128, dtype=F16, device=gpu)
        pool[pages - n:] = y[i]
        y[i] = pool
    y[3], y[6] = y[3] + (pages - n), y[6] + (pages - n)
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    got = impl_hip.run(*y)
    torch.cuda.synchronize()
    check(got, x)


def test_more_rows_than_a_launch_has_wavefronts(gpu):
    """17 million rows: the combining wavefronts take several each."""
    _say("attention of 17 million rows")
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    B, Hq = 270001, 64
    x = make([1] * 50, [1 + i % 3 for i in range(50)], prefix=[40], Hq=Hq, Hkv=8, page=16, seed=17)
    y = _to(x, gpu)
    rows = torch.arange(B, device=gpu) % 50
    q = torch.randn(B, Hq, 64, device=gpu, dtype=F16)
    y[0], y[5], y[6], y[7] = q, torch.tensor([0, B], device=gpu).int(), y[6][rows], y[7][rows]
    y[8] = torch.arange(B + 1, device=gpu).int()
    out, lse = impl_hip.run(*y)
    torch.cuda.synchronize()
    for at in (0, 131000, B - 50):
        at = at // 50 * 50
        z = list(x)
        z[0] = q[at:at + 50].cpu()
        check((out[at:at + 50], lse[at:at + 50]), z)
    assert bool((lse[:, :] != 0).all()) and bool(out.isfinite().all())


def test_replays_streams_and_overlapping_calls(gpu):
    """A captured call replayed with new contents; calls on two streams at once."""
    _say("attention graph and streams")
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    kw = dict(n_q=[1] * 20 + [40], lens=[30] * 20 + [50], prefix=[2000], Hq=8, Hkv=2, D=128, page=64)
    x = _to(make(**kw, seed=11), gpu)
    impl_hip.run(*x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = impl_hip.run(*x)
    for seed in range(3):
        new = _to(make(**kw, seed=60 + seed), gpu)
        new[7] -= seed                                    # other lengths, the same tables
        for a, b in zip(x, new):
            if isinstance(a, torch.Tensor):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = impl_hip.run(*new)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [_to(make(**kw, seed=70 + i), gpu) for i in range(2)]
    want = [impl_hip.run(*v) for v in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, v in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(impl_hip.run(*v))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_queries(gpu):
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    x = _to(make([0, 0], [5, 6], prefix=[3], seed=1), gpu)
    out, lse = impl_hip.run(*x)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


@pytest.mark.parametrize("case", [0, 3, 10])
def test_engine_drives_the_operator(gpu, case):
    from tilebench_amd.core import engine

    _say("engine", case)
    rows = engine.run_benchmark_suite("shared_prefix_attention", benchmark_overrides={"case_indices": [case], "repeat": 1},
                                      enabled_backends=["hip"])
    assert len(rows) == 1 and rows[0]["hip_ok"], rows[0]["hip_err"]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_a_layer_s_attention_path(gpu, cache):
    """As a served layer runs it: W4A16 QKV projection, append with the rotation,
    attention over the cache, W4A16 output projection; a prompt chunk, then
    decoded tokens.  Against the torch references of the same steps."""
    from tilebench_amd.benchmarks.operators.w4a16_gemm import impl_hip as linear
    from tilebench_amd.benchmarks.operators.w4a16_gemm import impl_torch as linear_ref
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip as append
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_torch as append_ref
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip as attend
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_torch as attend_ref

    _say("layer", cache)
    H, Hq, Hkv, D, P, B, prefix = 512, 8, 2, 64, 16, 3, 50
    g = torch.Generator().manual_seed(21)
    qkv = [t.to(gpu) for t in T.random_int4_weights(H, (Hq + 2 * Hkv) * D, 128, g)]
    proj = [t.to(gpu) for t in T.random_int4_weights(Hq * D, H, 128, g)]
    pools = T.paged_cache(40, Hkv, P, D, F16, g, cache == "e4m3", gpu)
    ref_pools = [c.clone() for c in pools]
    inv_freq, axes = (t.to(gpu) for t in T.rotary_frequencies(D, 1, 10000.0))
    order = torch.randperm(40, generator=g).int()
    pp, pages = order[:4].view(1, 4), order[4:4 + B * 4].view(B, 4)
    pl, go = torch.tensor([prefix]).int(), torch.tensor([0, B]).int()
    own = [0] * B
    for n_q in ([9, 20, 1], [1, 1, 1], [1, 2, 1]):
        own = [a + b for a, b in zip(own, n_q)]
        cu = [sum(n_q[:i]) for i in range(B + 1)]
        at = [(b, own[b] - n_q[b] + i) for b in range(B) for i in range(n_q[b])]
        positions = torch.tensor([prefix + j for _, j in at]).int().to(gpu)
        slots = torch.tensor([int(pages[b, j // P]) * P + j % P for b, j in at]).int().to(gpu)
        X = torch.randn(cu[-1], H, generator=g).half().to(gpu)
        y = linear.run(X, *qkv, 128).view(cu[-1], -1, D)
        yr = linear_ref.run(X, *qkv, 128).view(cu[-1], -1, D)
        tables = [t.to(gpu) for t in (pp, pl, go, pages, torch.tensor(own).int(), torch.tensor(cu).int())]
        q, *_ = append.run(y[:, :Hq], y[:, Hq:Hq + Hkv], y[:, Hq + Hkv:], positions, inv_freq, axes, slots, *pools)
        qr, *ref_pools = append_ref.run(yr[:, :Hq], yr[:, Hq:Hq + Hkv], yr[:, Hq + Hkv:], positions, inv_freq, axes,
                                        slots, *ref_pools)
        out, _ = attend.run(q, *pools[:2], *tables, max(n_q), None, *pools[2:])
        outr, _ = attend_ref.run(qr, *ref_pools[:2], *tables, max(n_q), None, *ref_pools[2:])
        z = linear.run(out.reshape(cu[-1], Hq * D), *proj, 128)
        zr = linear_ref.run(outr.reshape(cu[-1], Hq * D), *proj, 128)
        torch.cuda.synchronize()
        # the linear layers agree within 1e-2; an e4m3 code may differ by one step (1/8) where they differ
        torch.testing.assert_close(out.float(), outr.float(), rtol=5e-2, atol=5e-2 * float(outr.float().abs().max()))
        torch.testing.assert_close(z.float(), zr.float(), rtol=5e-2, atol=5e-2 * float(zr.float().abs().max()))
