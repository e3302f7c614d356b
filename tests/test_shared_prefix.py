"""Shared-prefix attention on the host: the torch reference against the formula row
by row, and what the operator refuses before any device is touched."""
import ctypes
import math

import pytest
import torch

from tests.shared_prefix_cases import make, reference
from tilebench_amd import paged
from tilebench_amd import runtime as rt


def by_row(x):
    """Every row by itself from the formula, fp64."""
    q, kc, vc, pp, pl, go, pages, lens, cu, max_q, scale = x[:11]
    ks, vs = (x[11], x[12]) if len(x) > 11 else (None, None)
    T, Hq, D = q.shape
    N, Hkv, P, _ = kc.shape
    out, lse = torch.zeros(T, Hq, D, dtype=torch.float64), torch.full((T, Hq), -math.inf, dtype=torch.float64)

    def token(c, s, ids, j, h):
        page = min(max(int(ids[j // P]), 0), N - 1)
        v = c[page, h, j % P].double()
        return v if s is None else v * float(s[page, h, j % P])

    for b in range(len(lens)):
        g = 0 if pp is None else max(i for i in range(pp.shape[0]) if int(go[i]) <= b)
        n = 0 if pp is None else int(pl[g])
        n_q, own = int(cu[b + 1] - cu[b]), int(lens[b])
        for i in range(n_q):
            see = [(pp[g], j) for j in range(n)] + [(pages[b], j) for j in range(own)]
            see = see[:max(n + own - n_q + i + 1, 0)]
            for hq in range(Hq):
                h = hq // (Hq // Hkv)
                if not see:
                    continue
                qq = q[int(cu[b]) + i, hq].double()
                s = torch.stack([token(kc, ks, ids, j, h) @ qq for ids, j in see]) * (D ** -0.5 if scale is None else scale)
                v = torch.stack([token(vc, vs, ids, j, h) for ids, j in see])
                out[int(cu[b]) + i, hq] = torch.softmax(s, dim=0) @ v
                lse[int(cu[b]) + i, hq] = torch.logsumexp(s, dim=0)
    return out, lse


@pytest.mark.parametrize("kw", [
    dict(n_q=[1, 1, 1], lens=[3, 17, 1]),
    dict(n_q=[1, 2, 0, 5], lens=[3, 9, 4, 5], prefix=[7, 0], bounds=[0, 2, 4], page=4, pad=2, spare=1),
    dict(n_q=[3, 1], lens=[1, 0], prefix=[1], page=2, cache="e4m3", dtype=torch.bfloat16),   # queries before the tokens
    dict(n_q=[2, 1], lens=[0, 0], page=8),                                                   # rows that see nothing
])
def test_reference_is_the_formula(kw):
    x = make(**kw, Hq=4, Hkv=2, D=64, seed=3)
    out, lse, _ = reference(x)
    want, want_lse = by_row(x)
    torch.testing.assert_close(out, want, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(lse, want_lse, rtol=1e-12, atol=1e-12)


@pytest.fixture
def impl():
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    from tilebench_amd.benchmarks.serving.shared_prefix_attention import impl_hip

    return impl_hip


@pytest.mark.parametrize("at,value,error", [
    (0, lambda v: v[0], ValueError), (0, lambda v: v.float(), TypeError), (0, lambda v: v[:, :3], ValueError),
    (0, lambda v: v[:, :, :32], ValueError), (1, lambda v: v[:, :1], ValueError), (1, lambda v: v.bfloat16(), TypeError),
    (3, lambda v: None, ValueError), (3, lambda v: v.long(), TypeError), (3, lambda v: v[0], ValueError),
    (3, lambda v: v[:, :0], ValueError), (4, lambda v: v.repeat(3), ValueError), (5, lambda v: v[:1], ValueError),
    (6, lambda v: v.long(), TypeError), (6, lambda v: v[:, :0], ValueError), (7, lambda v: v[:1], ValueError),
    (8, lambda v: v[:1], ValueError), (8, lambda v: v.long(), TypeError), (9, lambda v: -1, ValueError),
])
def test_refusals(impl, at, value, error):
    x = make([1, 2], [3, 40], prefix=[20], seed=1)
    assert impl.check(*x) == (3, 8, 2, 64, 1, 2, 2, 3, 6, 16)
    x[at] = value(x[at])
    with pytest.raises(error, match="shared_prefix_attention"):
        impl.check(*x)


def test_refusals_of_caches(impl):
    x = make([1], [3], seed=1)
    odd = torch.zeros(1, 2, 16, 72, dtype=torch.float16)[..., :64]       # rows of 144 bytes are 16-byte aligned
    assert impl.check(x[0], odd, odd, *x[3:])
    for width, shift in ((68, 0), (80, 4)):                               # rows of 136 bytes; rows that start 8 bytes off
        bad = torch.zeros(1, 2, 16, width, dtype=torch.float16)[..., shift:shift + 64]
        with pytest.raises(ValueError, match="16-byte"):
            impl.check(x[0], bad, bad, *x[3:])
    y = make([1], [3], Hq=4, Hkv=2, D=128, seed=1)
    y[0] = y[0][:, :, :96]
    c = [t[..., :96].contiguous() for t in y[1:3]]
    with pytest.raises(ValueError, match="64 or 128"):
        impl.check(y[0], *c, *y[3:])


def test_entry_point_checks_before_touching_a_device():
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    lib, fake = rt.load_library(), 1 << 40
    base = dict(q=fake, kc=fake, ks=None, pp=fake, cu=fake, T=8, Hq=8, Hkv=2, D=64, G=1, Wp=90, B=2, W=4, max_q=4, N=16,
                P=16, q_st=512, c_slot=64, scale=0.125, dtype=1, cache=1, ws=None, wb=0)

    def attend(**kw):
        a = {**base, **kw}
        return lib.tb_shared_prefix_attention(
            a["q"], a["kc"], fake, a["ks"], a["ks"], a["pp"], fake, fake, fake, fake, a["cu"], fake, fake, a["T"],
            a["Hq"], a["Hkv"], a["D"], a["G"], a["Wp"], a["B"], a["W"], a["max_q"], a["N"], a["P"], a["q_st"], 64, 2048,
            1024, a["c_slot"], 0, 0, 0, a["scale"], a["dtype"], a["cache"], a["ws"], a["wb"], None)

    for kw in (dict(T=-1), dict(Hq=7), dict(Hkv=0), dict(D=96), dict(P=12), dict(P=8192), dict(G=0), dict(Wp=0),
               dict(B=0), dict(W=0), dict(dtype=0), dict(cache=2), dict(cache=3), dict(ks=fake), dict(N=0),
               dict(N=1 << 30), dict(q=None), dict(pp=None), dict(cu=None), dict(q_st=510), dict(c_slot=60),
               dict(T=1 << 30), dict(W=1 << 28), dict(max_q=-1), dict(T=1 << 61), dict(max_q=1 << 61), dict(B=1 << 61),
               dict(scale=float("nan")), dict(scale=float("-inf")), dict(scale=1e39)):
        assert attend(**kw) == rt.TB_E_INVALID, kw
        assert "tb_shared_prefix_attention" in lib.tb_last_error().decode()
    assert attend(q=fake + 8) == rt.TB_E_ALIGN and attend(kc=fake + 8) == rt.TB_E_ALIGN
    assert attend(T=0) == rt.TB_OK                                   # nothing to do, nothing launched
    assert attend() == rt.TB_E_WORKSPACE and "workspace" in lib.tb_last_error().decode()
    need = ctypes.c_int64(-1)
    size = lib.tb_shared_prefix_attention_workspace_size
    assert size(8, 8, 2, 64, 1, 90, 2, 4, 16, 4, 1, ctypes.byref(need)) == rt.TB_OK and need.value > 0
    assert attend(ws=fake, wb=need.value - 1) == rt.TB_E_WORKSPACE
    assert attend(ws=fake + 4, wb=need.value) == rt.TB_E_ALIGN
    assert size(0, 8, 2, 64, 1, 4, 2, 4, 16, 4, 1, ctypes.byref(need)) == rt.TB_OK and need.value == 0
    # no prefix, and enough sequences to fill the device without splits: written directly
    assert size(512, 8, 8, 64, 0, 0, 512, 64, 16, 1, 1, ctypes.byref(need)) == rt.TB_OK and need.value == 0
    # short prefixes: every sequence reads its own
    assert size(8, 8, 2, 64, 1, 4, 2, 4, 16, 4, 1, ctypes.byref(need)) == rt.TB_OK and need.value == 0
    assert size(8, 8, 2, 64, 1, 4, 2, 4, 16, 4, 1, None) == rt.TB_E_INVALID


@pytest.mark.parametrize("tokens,heads", [(1, 8), (1, 1), (3, 1), (3, 8)])
@pytest.mark.parametrize("shift,gap", [(0, 3), (3, 0), (8, 8), (3, 5)])
def test_queries_of_any_layout_are_taken(tokens, heads, shift, gap):
    """Slices of a wider projection, one token or one head of it among them, whose row stride PyTorch keeps in copies."""
    wide = torch.randn(tokens + 1, heads * 64 + shift + gap, generator=torch.Generator().manual_seed(1)).half()
    x = wide[:, shift:shift + heads * 64].view(tokens + 1, heads, 64)[1:]
    y = paged.aligned_rows(x, 8)
    assert torch.equal(y, x) and y.data_ptr() % 16 == 0 and y.stride(-1) == 1
    assert all(s % 8 == 0 for s in y.stride()[:-1])
    fine = x.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in x.stride()[:-1])
    assert (y.data_ptr() == x.data_ptr()) == fine                           # copied only where it has to be
    last = torch.empty(tokens, 64, heads).half().transpose(1, 2)            # the last dimension strided
    assert paged.aligned_rows(last, 8).stride(-1) == 1


MIB = 1 << 20


@pytest.mark.parametrize("kw", [
    dict(T=16384, Hq=64, Hkv=8, W=256, B=1, max_q=16384),                        # one long prompt
    dict(T=131072, Hq=64, Hkv=8, W=2048, B=1, max_q=131072),
    dict(T=8192, Hq=64, Hkv=8, W=64, B=16, max_q=512, G=1, Wp=94),               # prompts behind a cached one
    dict(T=32768, Hq=64, Hkv=8, W=64, B=64, max_q=512, G=4, Wp=94),
    dict(T=4385, Hq=32, Hkv=8, W=15, B=16, max_q=500, G=1, Wp=94),
    dict(T=40000, Hq=32, Hkv=8, W=64, B=10000, max_q=4000, G=1, Wp=94),          # one prompt among many decodes
    dict(T=300, Hq=32, Hkv=8, W=64, B=300, max_q=1, G=300, Wp=2048),             # a group for each sequence
    dict(T=10000, Hq=32, Hkv=8, W=2048, B=10000, max_q=1, G=10000, Wp=2048),
    dict(T=4096, Hq=64, Hkv=8, W=2048, B=4096, max_q=1, G=1, Wp=128),
    dict(T=270001, Hq=64, Hkv=8, D=64, W=1, B=270001, max_q=1, G=1, Wp=3, page=16),
])
@pytest.mark.parametrize("cache", [1, 3])
def test_workspaces_are_bounded(kw, cache):
    """Results of what tiles split, five of every row that streams may work on or 640 MiB of them, 16 bytes a row."""
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    c = {**dict(D=128, G=0, Wp=0, page=64), **kw}
    need = ctypes.c_int64(-1)
    size = rt.load_library().tb_shared_prefix_attention_workspace_size
    args = [c[k] for k in ("T", "Hq", "Hkv", "D", "G", "Wp", "B", "W", "page", "max_q")]
    assert size(*args, cache, ctypes.byref(need)) == rt.TB_OK
    rows, each = c["T"] * c["Hq"], c["D"] * 4 + 8
    prompts = c["max_q"] * c["Hq"] // c["Hkv"] > 16   # then streams take sequences of up to 16 rows a key/value head
    few = min(rows, c["B"] * c["Hkv"] * 16) if prompts else rows
    assert 0 <= need.value <= max(5 * few * each, 640 * MIB) + 72 * MIB + 16 * rows, need.value / MIB
    if few <= 16384:
        assert need.value <= 512 * MIB


def test_limits_of_sizes_are_the_documented_ones():
    """The largest sizes that the header allows are taken, one more is refused by name."""
    if not rt.LIB_PATH.exists():
        pytest.skip("libtbhip.so is not built")
    lib, need = rt.load_library(), ctypes.c_int64(-1)

    def size(T=8, Hq=8, Hkv=8, G=1, Wp=1, B=1, W=1, page=64, max_q=1):
        return lib.tb_shared_prefix_attention_workspace_size(T, Hq, Hkv, 64, G, Wp, B, W, page, max_q, 1,
                                                             ctypes.byref(need))

    table = 2 ** 29 // 64
    for fits, over in ((dict(T=2 ** 28 - 1), dict(T=2 ** 28)), (dict(max_q=2 ** 28 - 1), dict(max_q=2 ** 28)),
                       (dict(B=2 ** 20 - 1), dict(B=2 ** 20)), (dict(G=2 ** 20 - 1), dict(G=2 ** 20)),
                       (dict(Wp=table - 1), dict(Wp=table)), (dict(W=table - 1, Hkv=1, Hq=1), dict(W=table, Hkv=1, Hq=1))):
        assert size(**fits) == rt.TB_OK, fits
        assert size(**over) == rt.TB_E_INVALID and "2^31" in lib.tb_last_error().decode(), over
    # sequences, key/value heads and steps of 32 tokens: 2^30 at most
    assert size(B=2 ** 16, W=2 ** 10) == rt.TB_OK
    assert size(B=2 ** 16, W=2 ** 10 + 1) == rt.TB_E_INVALID
    assert "65536 sequences" in lib.tb_last_error().decode() and "2^30" in lib.tb_last_error().decode()
