"""Rotary positions and cache appends on the host: the torch references against
the definition in 64 bits, the gradient against differences, and what the
operators refuse (checked before any device is touched)."""
import numpy as np
import pytest
import torch

from tilebench_amd import paged
from tilebench_amd import runtime as rt
from tilebench_amd.benchmarks.serving.rope_kv_append import impl_torch as append_ref
from tilebench_amd.benchmarks.serving.rotary_axes import impl_torch as rotary_ref
from tilebench_amd.data import tensors as T
from tilebench_amd.paths import list_operators, list_serving_operators, operator_config, operator_package


def definition(x, positions, inv_freq, axes, interleaved, sign=1.0):
    """The rotation as products of complex numbers, fp64 numpy."""
    x = x.double().numpy()
    P = inv_freq.numel()
    pos = positions.numpy().reshape(-1, x.shape[0]).astype(np.float64)
    ax = np.zeros(P, int) if axes is None else axes.numpy()
    turn = np.exp(1j * sign * pos[ax].T * inv_freq.double().numpy())[:, None]
    out = x.copy()
    if interleaved:
        z = (x[..., 0:2 * P:2] + 1j * x[..., 1:2 * P:2]) * turn
        out[..., 0:2 * P:2], out[..., 1:2 * P:2] = z.real, z.imag
    else:
        z = (x[..., :P] + 1j * x[..., P:2 * P]) * turn
        out[..., :P], out[..., P:2 * P] = z.real, z.imag
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,axes", [(8, 8, 1), (12, 6, 3), (80, 80, 2), (128, 64, 3)])
def test_reference_is_the_definition(D, R, axes, interleaved):
    g = torch.Generator().manual_seed(D + axes)
    q, k = torch.randn(5, 3, D, generator=g), torch.randn(5, 1, D, generator=g)
    positions = torch.randint(-100000, 100000, (axes, 5), generator=g).int()
    inv_freq, ax = T.rotary_frequencies(R, axes, 10000.0)
    out = rotary_ref.run(q, k, positions, inv_freq, ax, interleaved)
    for x, y in zip((q, k), out):
        # cos and sin rounded to fp32 (2^-24 each), two products and a sum: under 4 roundings of values up to |a| + |b|
        bound = 4 * 2.0 ** -24 * 2 * float(x.abs().max())
        np.testing.assert_allclose(y.double().numpy(), definition(x, positions, inv_freq, ax, interleaved), rtol=0,
                                   atol=bound)
    back = rotary_ref.run(*out, positions, inv_freq, ax, interleaved, inverse=True)
    np.testing.assert_allclose(back[0].numpy(), q.numpy(), rtol=0, atol=16 * 2.0 ** -24 * 2 * float(q.abs().max()))


def test_gradient_is_the_inverse_rotation_by_differences():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(3, 2, 8, generator=g), torch.randn(3, 2, 8, generator=g)
    positions = torch.tensor([[0, 7, 1000], [3, 2, 1]], dtype=torch.int32)
    inv_freq, ax = T.rotary_frequencies(8, 2, 100.0)
    for interleaved in (False, True):
        grad = rotary_ref.run(w, None, positions, inv_freq, ax, interleaved, inverse=True)[0].double().numpy()
        xd = x.double()
        h = 1e-3
        for i in np.ndindex(3, 2, 8):
            up, down = xd.clone(), xd.clone()
            up[i] += h
            down[i] -= h
            f = [float((definition(v, positions, inv_freq, ax, interleaved) * w.double().numpy()).sum())
                 for v in (up, down)]
            # linear in x: the central difference is exact up to fp64; the gradient carries four fp32 roundings
            assert abs((f[0] - f[1]) / (2 * h) - grad[i]) < 4 * 2.0 ** -24 * 2 * float(w.abs().max()) + 1e-9


def test_append_reference_writes_the_named_slots_only():
    q, k, v, pos, f, ax, slots, kc, vc, ks, vs = T.generate_rope_kv_append_inputs(
        6, Hq=2, Hkv=1, D=16, page=4, cache="e4m3", seed=3, device="cpu")
    slots[2], slots[4] = -1, kc.shape[0] * 4
    k[0], v[1] = 0, 0
    out = append_ref.run(q, k, v, pos, f, ax, slots, kc, vc, ks, vs)
    written = set(int(s) for s in slots if 0 <= int(s) < kc.shape[0] * 4)
    rotated = rotary_ref.rotate(k, *rotary_ref.table(pos, f, ax))
    for new, old, scale, old_scale, x in ((out[1], kc, out[3], ks, rotated), (out[2], vc, out[4], vs, v.float())):
        for slot in range(kc.shape[0] * 4):
            page, at = divmod(slot, 4)
            if slot not in written:
                assert torch.equal(new[page, :, at].view(torch.uint8), old[page, :, at].view(torch.uint8))
                assert torch.equal(scale[page, :, at], old_scale[page, :, at])
                continue
            t = int((slots == slot).nonzero()[0])
            s = scale[page, :, at]
            assert torch.equal(s, x[t].abs().amax(dim=-1) / 448.0)
            back = new[page, :, at].float() * s[:, None]
            # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normals
            assert bool(((back - x[t]).abs() <= 2.0 ** -4 * x[t].abs() * (1 + 1e-6) + 2.0 ** -10 * s[:, None]).all())


def test_serving_operators_are_registered_beside_the_others():
    import yaml

    ops = list_serving_operators()
    assert {"rotary_axes", "rope_kv_append"} <= set(ops) and not set(ops) & set(list_operators())
    assert operator_package("int4_dequant") == "tilebench_amd.benchmarks.operators.int4_dequant"
    for op in ops:
        assert operator_package(op) == f"tilebench_amd.benchmarks.serving.{op}"
        cfg = yaml.safe_load(open(operator_config(op)))
        assert T.expand_cases(op, cfg) and T.get_generator(op) is not None
        assert cfg["benchmark"]["warmup"] == 1 and cfg["benchmark"]["repeat"] == 3


# ----------------------------------------------------------------------------- refusals


def _rotation(Tn=4, Hq=2, Hk=1, D=16, R=16, axes=1, dtype=torch.float16):
    f, ax = T.rotary_frequencies(R, axes, 10000.0)
    return [torch.zeros(Tn, Hq, D, dtype=dtype), torch.zeros(Tn, Hk, D, dtype=dtype),
            torch.zeros(axes, Tn, dtype=torch.int32), f, ax]


@pytest.mark.parametrize("change,error", [
    (lambda x: x.__setitem__(0, x[0][0]), ValueError),                              # q of two dimensions
    (lambda x: x.__setitem__(1, torch.zeros(5, 1, 16).half()), ValueError),         # other tokens
    (lambda x: x.__setitem__(1, torch.zeros(4, 1, 8).half()), ValueError),          # other head dimension
    (lambda x: x.__setitem__(1, x[1].bfloat16()), TypeError),                       # mixed types
    (lambda x: x.__setitem__(0, x[0].double()), TypeError),
    (lambda x: x.__setitem__(2, x[2].long()), TypeError),                           # int64 positions
    (lambda x: x.__setitem__(2, x[2][:, :3]), ValueError),                          # positions of other tokens
    (lambda x: x.__setitem__(2, torch.zeros(9, 4, dtype=torch.int32)), ValueError),  # nine axes
    (lambda x: x.__setitem__(3, x[3].double()), TypeError),
    (lambda x: x.__setitem__(3, torch.zeros(9)), ValueError),                       # more pairs than channels
    (lambda x: x.__setitem__(3, torch.zeros(0)), ValueError),
    (lambda x: x.__setitem__(4, x[4].long()), TypeError),
    (lambda x: x.__setitem__(4, x[4][:3]), ValueError),
    (lambda x: (x.__setitem__(2, x[2].expand(2, 4)), x.__setitem__(4, None)), ValueError),  # two axes, no map
])
def test_rotation_refusals(change, error):
    x = _rotation()
    paged.check_rotation("op", *x)
    change(x)
    with pytest.raises(error, match="op"):
        paged.check_rotation("op", *x)


@pytest.mark.parametrize("change,error", [
    (lambda c: c.update(k=c["k"][:, :, :, :8]), ValueError),
    (lambda c: c.update(v=c["v"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)), ValueError),  # other strides
    (lambda c: c.update(k=c["k"].bfloat16(), v=c["v"].bfloat16()), TypeError),
    (lambda c: c.update(heads=3), ValueError),
    (lambda c: c.update(k=c["k"][:, :, :3], v=c["v"][:, :, :3]), ValueError),      # page of three slots
    (lambda c: c.update(k=c["k"][:0], v=c["v"][:0]), ValueError),                  # no pages
    (lambda c: c.update(k=c["k"][:1].expand(4, 2, 4, 16), v=c["v"][:1].expand(4, 2, 4, 16)), ValueError),
    (lambda c: c.update(k=c["k"].transpose(2, 3), v=c["v"].transpose(2, 3), D=4), ValueError),
    (lambda c: c.update(ks=torch.zeros(4, 2, 4)), ValueError),                     # scales of a 16-bit cache
    (lambda c: c.update(k=c["k"].to(torch.float8_e4m3fn), v=c["v"].to(torch.float8_e4m3fn)), ValueError),
    (lambda c: c.update(k=c["k"].to(torch.float8_e4m3fn), v=c["v"].to(torch.float8_e4m3fn),
                        ks=torch.zeros(4, 2, 4).half(), vs=torch.zeros(4, 2, 4).half()), TypeError),
    (lambda c: c.update(k=c["k"].to(torch.float8_e4m3fn), v=c["v"].to(torch.float8_e4m3fn),
                        ks=torch.zeros(4, 4, 2), vs=torch.zeros(4, 4, 2)), ValueError),
])
def test_cache_refusals(change, error):
    c = dict(heads=2, D=16, k=torch.zeros(4, 2, 4, 16).half(), v=torch.zeros(4, 2, 4, 16).half(), ks=None, vs=None)
    call = lambda: paged.check_cache("op", torch.float16, c["heads"], c["D"], c["k"], c["v"], c["ks"], c["vs"])  # noqa: E731
    assert call() == (4, 4)
    change(c)
    with pytest.raises(error, match="op"):
        call()


@pytest.mark.parametrize("at,value,error", [
    (0, lambda x: x.float(), TypeError), (2, lambda x: x[:, :, :8], ValueError), (2, lambda x: x.bfloat16(), TypeError),
    (2, lambda x: None, ValueError), (6, lambda x: x.long(), TypeError), (6, lambda x: x[:2], ValueError),
])
def test_append_refusals(at, value, error):
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    from tilebench_amd.benchmarks.serving.rope_kv_append import impl_hip

    x = list(T.generate_rope_kv_append_inputs(3, Hq=2, Hkv=1, D=16, page=4, device="cpu"))
    assert impl_hip.check(*x) == (3, 2, 1, 16, 16, 1, 5, 4)
    x[at] = value(x[at])
    if at == 0:
        x[1] = value(x[1])
    with pytest.raises(error, match="rope_kv_append"):
        impl_hip.check(*x)


def test_entry_points_check_before_touching_a_device():
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    lib, fake = rt.load_library(), 1 << 40

    def rotary(T=4, Hq=2, Hk=1, D=16, R=16, A=1, q=fake, k=fake, axes=fake, dtype=1):
        return lib.tb_rotary_axes(q, fake, k, fake, fake, fake, axes, T, Hq, Hk, D, R, A, 32, 16, 16, 16, dtype, 0, 0,
                                  None)

    def append(T=4, Hkv=1, D=16, pages=4, page=4, dtype=1, cache=1, scale=None):
        return lib.tb_rope_kv_append(fake, fake, fake, fake, fake, fake, fake, fake, fake, fake, scale, scale, T, 2,
                                     Hkv, D, 16, 1, 32, 16, 16, 16, 16, 16, pages, page, 64, 64, 16, 4, 4, 1, dtype,
                                     cache, 0, None)

    for kw in (dict(q=None), dict(k=None), dict(D=15), dict(D=514), dict(R=18), dict(R=0), dict(A=0), dict(A=9),
               dict(A=2, axes=None), dict(dtype=3), dict(T=-1), dict(Hq=0)):
        assert rotary(**kw) == rt.TB_E_INVALID, kw
        assert "tb_rotary_axes" in lib.tb_last_error().decode()
    assert rotary(T=0) == rt.TB_OK and append(T=0) == rt.TB_OK      # nothing to do, nothing launched
    for kw in (dict(Hkv=0), dict(page=3), dict(page=8192), dict(pages=0), dict(pages=1 << 30), dict(dtype=0),
               dict(cache=2), dict(cache=3), dict(scale=fake)):
        assert append(**kw) == rt.TB_E_INVALID, kw
        assert "tb_rope_kv_append" in lib.tb_last_error().decode()


def test_caches_of_one_head_or_page_in_either_order():
    """Strides of dimensions of size 1 say nothing: [pages, page, 1, D] pools beside [pages, 1, page, D] ones."""
    for pages, heads, page in ((4, 1, 8), (1, 2, 8), (1, 1, 1), (4, 2, 1)):
        k = torch.zeros(pages, heads, page, 16).half()
        v = torch.zeros(pages, page, heads, 16).half().permute(0, 2, 1, 3)
        if heads > 1 and page > 1:
            v = torch.zeros(pages + 1, 3, heads, page, 16).half()[1:, 1]      # one page of a wider pool
        assert pages > 1 and page == 1 or v.stride() != k.stride() or k.numel() == 16
        assert paged.check_cache("op", torch.float16, heads, 16, k, v, None, None) == (pages, page)
        c = k.to(torch.float8_e4m3fn)
        scales = torch.zeros(pages, heads, page), torch.zeros(pages, page, heads).transpose(1, 2)
        if heads > 1 and page > 1:
            scales = scales[0], torch.zeros(pages + 1, 3, heads, page)[1:, 1]
        assert paged.check_cache("op", torch.float16, heads, 16, c, c, *scales) == (pages, page)
    one = torch.zeros(4, 1, 1, 16).half().expand(4, 1, 8, 16)                 # but no dimension may be expanded
    with pytest.raises(ValueError, match="expanded"):
        paged.check_cache("op", torch.float16, 1, 16, one, one, None, None)
