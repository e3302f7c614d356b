"""Rotary positions with several axes and appends to a paged cache on the GPU,
against the definition in 64 bits on the CPU.

Tolerances.  A result is p * c - q * s with c and s rounded once to fp32 (and
the reduced angle too: 2^-25 turns of error, 2e-7 rad), two products and a sum
in fp32, and one rounding to the type: 2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32) of
the value, half the smallest subnormal at least, plus 8 * 2^-24 * (|p| + |q|)."""
import numpy as np
import pytest
import torch

from tests.test_rotary import definition
from tilebench_amd.data import tensors as T

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _say(*a):
    print("[gpu case]", *a, flush=True)


def _close(y, want, x, dtype):
    """y of `dtype` against fp64 `want`, inputs as large as x."""
    y = y.detach().cpu().double().numpy()
    err = np.abs(y - want)
    bound = HALF[dtype] * np.abs(want) * (1 + 1e-6) + TINY[dtype] + 8 * 2.0 ** -24 * 2 * float(x.abs().max())
    assert (err <= bound).all(), float((err - bound).max())


def _rotary(q, k, pos, f, ax, gpu, **kw):
    from tilebench_amd.benchmarks.serving.rotary_axes import impl_hip

    out = impl_hip.run(*(None if x is None else x.to(gpu) for x in (q, k, pos, f, ax)), **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("Tn,Hq,Hk,D,R,axes,interleaved,dtype", [
    (1, 1, 1, 2, 2, 1, False, "fp16"), (1, 32, 8, 128, 128, 1, False, "bf16"), (3, 5, 1, 80, 80, 2, False, "bf16"),
    (7, 4, 2, 72, 72, 2, False, "fp16"), (7, 4, 2, 72, 72, 2, True, "fp16"), (33, 3, 3, 6, 4, 3, False, "fp32"),
    (33, 3, 3, 6, 4, 3, True, "bf16"), (129, 8, 8, 128, 64, 3, True, "fp32"), (129, 8, 8, 128, 64, 3, False, "fp16"),
    (50, 2, 1, 512, 512, 4, False, "bf16"), (50, 2, 1, 510, 34, 8, True, "fp16"), (12, 2, 1, 96, 40, 2, False, "fp32"),
    (4097, 16, 4, 64, 64, 2, False, "fp16"), (1027, 32, 8, 128, 96, 3, True, "bf16"),
])
def test_rotary_matches_the_definition(gpu, Tn, Hq, Hk, D, R, axes, interleaved, dtype):
    _say("rotary", Tn, Hq, Hk, D, R, axes, interleaved, dtype)
    g = torch.Generator().manual_seed(Tn + D)
    q, k = (torch.randn(Tn, h, D, generator=g).to(DT[dtype]) for h in (Hq, Hk))
    pos = torch.randint(-200000, 200000, (axes, Tn), generator=g).int()
    f, ax = T.rotary_frequencies(R, axes, 10000.0)
    for inverse in (False, True):
        out = _rotary(q, k, pos, f, ax, gpu, interleaved=interleaved, inverse=inverse)
        for x, y in zip((q, k), out):
            assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
            _close(y, definition(x, pos, f, ax, interleaved, -1.0 if inverse else 1.0), x, DT[dtype])


def test_far_positions_keep_their_angles(gpu):
    """Angles of up to 2^31 rad: the 64-bit reduction leaves 2^31 * 2^-53 turns."""
    _say("rotary far positions")
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 12345678], dtype=torch.int32)
    q = torch.randn(4, 2, 16, generator=torch.Generator().manual_seed(1))
    f, ax = T.rotary_frequencies(16, 1, 10000.0)
    out = _rotary(q, None, pos, f, None, gpu)
    assert out[1] is None
    _close(out[0], definition(q, pos, f, None, False), q, torch.float32)


def test_strides_and_alignment_do_not_change_bits(gpu):
    """Views of a fused projection, heads before tokens, rows that start off a 16-byte
    border, an odd token stride and a strided last dimension give the dense call's bits."""
    _say("rotary strides")
    from tilebench_amd.benchmarks.serving.rotary_axes import impl_hip

    g = torch.Generator().manual_seed(5)
    Tn, H, D = 37, 4, 64
    dense = torch.randn(Tn, H, D, generator=g).half().to(gpu)
    f, ax = (x.to(gpu) for x in T.rotary_frequencies(D, 2, 10000.0))
    pos = torch.randint(0, 5000, (2, Tn), generator=g).int().to(gpu)
    want = impl_hip.run(dense, None, pos, f, ax)[0]
    wide = torch.zeros(Tn, H * D + 24, dtype=torch.float16, device=gpu)
    for shift in (8, 4, 1):
        view = wide[:, shift:shift + H * D].view(Tn, H, D)
        view.copy_(dense)
        assert torch.equal(impl_hip.run(view, None, pos, f, ax)[0], want), shift
    odd = torch.zeros(Tn, H * D + 1, dtype=torch.float16, device=gpu)[:, :H * D].view(Tn, H, D)
    odd.copy_(dense)
    heads_first = dense.transpose(0, 1).contiguous().transpose(0, 1)
    last = dense.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (odd, heads_first, last):
        assert torch.equal(impl_hip.run(x, None, pos, f, ax)[0], want)
    assert torch.equal(impl_hip.run(dense, dense, pos, f, ax)[1], want)   # one tensor as q and as k
    assert impl_hip.run(dense[:0], None, pos[:, :0], f, ax)[0].shape == (0, H, D)


def test_axes_outside_the_positions_are_clamped(gpu):
    _say("rotary axes clamped")
    g = torch.Generator().manual_seed(6)
    q = torch.randn(5, 2, 32, generator=g)
    pos = torch.randint(0, 100, (2, 5), generator=g).int()
    f, ax = T.rotary_frequencies(32, 2, 10000.0)
    wild = ax.clone()
    wild[0], wild[-1] = -7, 99
    assert torch.equal(_rotary(q, None, pos, f, wild, gpu)[0], _rotary(q, None, pos, f, ax, gpu)[0])


# ----------------------------------------------------------------------------- appends


def _append(x, gpu, **kw):
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

    y = [None if v is None else v.to(gpu) for v in x]
    out = impl_hip.run(*y, **kw)
    torch.cuda.synchronize()
    assert all(a is b for a, b in zip(out[1:], y[7:]))  # the caches given
    return out


def _check_append(x, out, interleaved=False):
    q, k, v, pos, f, ax, slots = x[:7]
    pools, scales = x[7:9], x[9:]
    P, total = pools[0].shape[2], pools[0].shape[0] * pools[0].shape[2]
    _close(out[0], definition(q, pos, f, ax, interleaved), q, q.dtype)
    keep = (slots >= 0) & (slots < total)
    at = slots[keep].long()
    for i, (rows, src) in enumerate(((definition(k, pos, f, ax, interleaved), k), (v.double().numpy(), v))):
        new, old = out[1 + i].cpu(), pools[i]
        touched = torch.zeros(total, dtype=torch.bool)
        touched[at] = True
        flat = lambda c: c.transpose(1, 2).reshape(total, *c.shape[1:2], *c.shape[3:])  # noqa: E731
        bits = lambda c: flat(c.view(torch.uint8 if c.element_size() == 1 else torch.int16))  # noqa: E731
        assert torch.equal(bits(new)[~touched], bits(old)[~touched])
        rows = rows[keep.numpy()]
        if not scales:
            _close(flat(new)[at], rows, src, src.dtype)
            continue
        s_new, s_old = flat(out[3 + i].cpu()), flat(scales[i])
        assert torch.equal(s_new[~touched], s_old[~touched])
        s, want = s_new[at].double().numpy(), np.abs(rows).max(axis=-1) / 448.0
        big = 2 * float(src.abs().max())
        # absmax of values that are off by 8 * 2^-24 * big, one rounding of the division
        assert (np.abs(s - want) <= 8 * 2.0 ** -24 * big / 448 + 2.0 ** -24 * want).all()
        back = flat(new)[at].float().double().numpy() * s[..., None]
        # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below the normals), the fp32 error before it,
        # and the same once more where that error crosses a border
        bound = 2.0 ** -4 * np.abs(rows) + 2.0 ** -10 * s[..., None] + 2 * 8 * 2.0 ** -24 * big
        assert (np.abs(back - rows) <= bound).all()


@pytest.mark.parametrize("Tn,Hq,Hkv,D,axes,page,cache,dtype,interleaved", [
    (1, 1, 1, 2, 1, 1, "same", "fp16", False), (1, 32, 8, 128, 1, 64, "same", "bf16", False),
    (1, 32, 8, 128, 1, 64, "e4m3", "fp16", False), (64, 8, 2, 64, 3, 16, "e4m3", "bf16", True),
    (64, 8, 2, 64, 3, 16, "same", "fp16", True), (77, 6, 3, 80, 2, 8, "e4m3", "fp16", False),
    (77, 6, 3, 72, 2, 8, "e4m3", "bf16", False), (77, 6, 3, 10, 2, 8, "e4m3", "bf16", True),
    (19, 2, 1, 512, 1, 4096, "e4m3", "fp16", False), (2500, 32, 8, 128, 3, 32, "same", "bf16", False),
    (2501, 32, 8, 128, 1, 128, "e4m3", "fp16", False),
])
def test_append_matches_the_definition(gpu, Tn, Hq, Hkv, D, axes, page, cache, dtype, interleaved):
    _say("append", Tn, Hq, Hkv, D, axes, page, cache, dtype, interleaved)
    x = T.generate_rope_kv_append_inputs(Tn, axes, Hq, Hkv, D, page, cache, dtype=DT[dtype], seed=Tn, device="cpu")
    if Tn > 3:
        x[6][1], x[6][Tn // 2] = -1, x[7].shape[0] * page   # padded tokens write nothing
    _check_append(x, _append(x, gpu, interleaved=interleaved), interleaved)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_append_into_pools_of_other_orders(gpu, cache):
    """[pages, page, heads, D] pools, and keys beside values in one allocation."""
    _say("append pool orders", cache)
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

    x = T.generate_rope_kv_append_inputs(40, 1, 8, 4, 64, 16, cache, seed=9, device="cpu")
    want = _append(x, gpu)
    y = [v.to(gpu) for v in x]
    u8 = lambda c: c.view(torch.uint8) if c.element_size() == 1 else c  # noqa: E731
    nhd = [u8(c).transpose(1, 2).contiguous().transpose(1, 2).view(c.dtype) for c in y[7:9]]
    both = torch.stack([u8(c) for c in y[7:9]], dim=1).contiguous()
    side = [both[:, i].view(y[7].dtype) for i in range(2)]
    sc = [s.transpose(1, 2).contiguous().transpose(1, 2) for s in y[9:]]
    for pools in (nhd, side):
        out = impl_hip.run(*y[:7], *pools, *[s.clone(memory_format=torch.preserve_format) for s in sc])
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(u8(a), u8(b))


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_keys_and_values_of_one_head_in_different_orders(gpu, cache):
    """With one head [pages, page, 1, D] and [pages, 1, page, D] are one order, whatever the strides say."""
    _say("append one head", cache)
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip as append
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip as attend

    y = [v.to(gpu) for v in T.generate_rope_kv_append_inputs(40, 1, 8, 1, 64, 16, cache, seed=9, device="cpu")]
    pools = [y[7].clone(), y[8].clone(), *(s.clone() for s in y[9:])]
    for i in range(1, len(pools), 2):
        x = pools[i].view(torch.uint8) if pools[i].element_size() == 1 else pools[i]
        other = x.new_empty(x.transpose(1, 2).shape).transpose(1, 2)
        pools[i] = other.copy_(x).view(pools[i].dtype)
        assert pools[i].stride() != pools[i - 1].stride()
    want, got = append.run(*y), append.run(*y[:7], *pools)
    tables = [torch.tensor(t, dtype=torch.int32, device=gpu) for t in ([[0, 1, 2]], [40], [0, 40])]
    a, b = (attend.run(x[0], *x[1:3], None, None, None, *tables, 40, None, *x[3:]) for x in (want, got))
    torch.cuda.synchronize()
    for u, v in zip((*want, *a), (*got, *b)):
        u, v = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (u, v))
        assert torch.equal(u, v)


def test_append_special_rows(gpu):
    """Zero rows (s = 0, codes 0), rows with inf and NaN (read back as NaN), next to ordinary heads."""
    _say("append special rows")
    x = T.generate_rope_kv_append_inputs(6, 1, 2, 2, 64, 8, "e4m3", seed=11, device="cpu")
    k, v, slots = x[1], x[2], x[6].long()
    k[0, 0], v[1, 1] = 0, 0
    v[2, 0, 5], v[3, 1, 63], k[4, 0, 7] = float("inf"), float("nan"), float("-inf")
    out = _append(x, gpu)
    at = slots // 8, slots % 8
    kc, vc, ks, vs = (c.cpu() for c in out[1:])
    kb, vb = (c[at[0], :, at[1]].float() * s[at[0], :, at[1]][..., None] for c, s in ((kc, ks), (vc, vs)))
    assert (kb[0, 0] == 0).all() and ks[at[0][0], 0, at[1][0]] == 0 and (vb[1, 1] == 0).all()
    assert vb[2, 0].isnan().all() and vb[3, 1].isnan().all() and kb[4, 0].isnan().all()
    bad = {(1, 2, 0), (1, 3, 1), (0, 4, 0)}
    for i, b in enumerate((kb, vb)):
        for t in range(6):
            for h in range(2):
                assert (i, t, h) in bad or b[t, h].isfinite().all()


def test_codes_are_rounded_as_by_division(gpu):
    """Rows of every magnitude: the scale absmax / 448 and the codes x * 448 / absmax, each rounded from 64 bits."""
    _say("append codes")
    x = list(T.generate_rope_kv_append_inputs(221, 1, 4, 4, 128, 16, "e4m3", dtype=torch.bfloat16, seed=3, device="cpu"))
    v = x[2].float() * 2.0 ** torch.arange(-120, 101).float()[:, None, None]
    x[2] = v.to(torch.bfloat16)
    out = _append(x, gpu)
    v, slots = x[2].float(), x[6].long()
    s = v.double().abs().amax(dim=-1) / 448.0
    code = (v / s[..., None]).float().to(torch.float8_e4m3fn)
    at = (slots // 16, slice(None), slots % 16)
    assert torch.equal(out[4].cpu()[at], s.float())
    assert torch.equal(out[2].cpu().view(torch.uint8)[at], code.view(torch.uint8))


def test_keys_are_quantised_as_in_64_bits(gpu):
    """Rotated keys' scales and codes are those of the definition in 64 bits, but for scales next to a border.

    Sine and cosine are off by at most 2^-36.5 (their series 2^-37 and 2^-41, the angle of up to 2^15.2 rad by 2^-37.8), a key by
    that times |a| + |b|, at most 2^0.5 times the row's largest: 2^-36 of the scale, half as much again for safety."""
    _say("append keys in 64 bits")
    x = T.generate_rope_kv_append_inputs(8192, 1, 8, 8, 128, 64, "e4m3", dtype=torch.bfloat16, seed=5, device="cpu")
    out = _append(x, gpu)
    rows, slots = definition(x[1], *x[3:6], False), x[6].long()
    at = (slots // 64, slice(None), slots % 64)
    want = np.abs(rows).max(axis=-1) / 448.0
    step = np.spacing(want.astype(np.float32)).astype(np.float64)
    away = np.abs(want / step - np.floor(want / step) - 0.5) * step > 1.5 * 2.0 ** -36 * want
    scales = out[3].cpu()[at].numpy()
    assert away.mean() > 0.99 and (scales == want.astype(np.float32))[away].all()
    codes = torch.from_numpy((rows / want[..., None]).astype(np.float32)).to(torch.float8_e4m3fn)
    assert torch.equal(out[1].cpu()[at].float(), codes.float())


def test_more_tokens_than_a_launch_has_wavefronts(gpu):
    """The tokens past 2^25 come in a second launch."""
    _say("rotary of 2^25 tokens")
    from tilebench_amd.benchmarks.serving.rotary_axes import impl_hip

    n = (1 << 25) + 5
    q = torch.randn(n, 1, 2, device=gpu, dtype=torch.float16)
    pos = torch.arange(n, device=gpu, dtype=torch.int32)
    f = torch.tensor([0.37])
    out, _ = impl_hip.run(q, None, pos, f.to(gpu))
    torch.cuda.synchronize()
    for a in (0, n // 2, (1 << 25) - 7):
        part = slice(a, a + 12)
        _close(out[part], definition(q[part].cpu(), pos[part].cpu()[None], f, None, False), q[part], torch.float16)
    # a rotation keeps lengths: two roundings to fp16 (2^-11 of each channel) and the angle's 2^-20
    a, b = q.double().norm(dim=-1), out.double().norm(dim=-1)
    assert bool(((a - b).abs() <= 2.0 ** -10 * a + 2.0 ** -20).all())


def test_append_past_4_gib_of_cache(gpu):
    """Offsets of more than 32 bits: rows at the end of a pool of 5 GiB a side."""
    _say("append 64-bit offsets")
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

    x = T.generate_rope_kv_append_inputs(3, 1, 8, 8, 128, 64, seed=12, device="cpu")
    pages = 5 * 2 ** 30 // (8 * 64 * 128 * 2)
    pools = [torch.zeros(pages, 8, 64, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
    slots = torch.tensor([pages * 64 - 1, (pages - 1) * 64, 5], dtype=torch.int32)
    y = [t.to(gpu) for t in x[:6]]
    impl_hip.run(*y, slots.to(gpu), *pools)
    torch.cuda.synchronize()
    want = definition(x[1], *x[3:6], False)
    got = torch.stack([pools[0][-1, :, 63], pools[0][-1, :, 0], pools[0][0, :, 5]])
    _close(got, want, x[1], torch.float16)
    assert torch.equal(torch.stack([pools[1][-1, :, 63], pools[1][-1, :, 0], pools[1][0, :, 5]]).cpu(), x[2])
    assert int((pools[1] != 0).any(dim=-1).sum()) == 24


def test_append_replayed_in_a_graph_and_on_a_side_stream(gpu):
    _say("append graph")
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

    x = [t.to(gpu) for t in T.generate_rope_kv_append_inputs(9, 1, 8, 2, 64, 16, "e4m3", seed=13, device="cpu")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        impl_hip.run(*x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = impl_hip.run(*x)
    for seed in range(3):
        new = [t.to(gpu) for t in T.generate_rope_kv_append_inputs(9, 1, 8, 2, 64, 16, "e4m3", seed=50 + seed,
                                                                   device="cpu")]
        for a, b in zip(x, new):
            (a.view(torch.uint8) if a.element_size() == 1 else a).copy_(
                b.view(torch.uint8) if b.element_size() == 1 else b)
        graph.replay()
        torch.cuda.synchronize()
        want = impl_hip.run(*new)
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a,
                               b.view(torch.uint8) if b.element_size() == 1 else b)


def test_host_tensors_are_refused(gpu):
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip as append
    from tilebench_amd.benchmarks.serving.rotary_axes import impl_hip as rotary

    x = T.generate_rope_kv_append_inputs(3, 1, 2, 1, 16, 4, seed=1, device="cpu")
    y = [t.to(gpu) for t in x]
    with pytest.raises(ValueError, match="is on cpu"):
        append.run(*y[:7], x[7], y[8])
    with pytest.raises(ValueError, match="is on cpu"):
        rotary.run(y[0], y[1], x[3], y[4], y[5])


@pytest.mark.parametrize("op", ["rotary_axes", "rope_kv_append"])
def test_engine_drives_the_operator(gpu, op):
    """run_bench's path: inputs, reference, verification and timing of a small case."""
    from tilebench_amd.core import engine

    _say("engine", op)
    rows = engine.run_benchmark_suite(op, benchmark_overrides={"case_indices": [0], "repeat": 1},
                                      enabled_backends=["hip"])
    assert len(rows) == 1 and rows[0]["hip_ok"], rows[0]["hip_err"]
    assert rows[0]["hip_ms"] > 0
