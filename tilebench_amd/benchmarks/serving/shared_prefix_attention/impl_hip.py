"""hip backend of paged attention over shared prefixes: tb_shared_prefix_attention in libtbhip.so.

run(q, k_cache, v_cache, prefix_pages, prefix_lens, group_offsets, pages, lens,
cu_q, max_q) returns (out [T, Hq, D], lse fp32 [T, Hq]).

q [T, Hq, D] holds the queries of B sequences, those of sequence b in rows
cu_q[b] .. cu_q[b + 1] - 1 (int32 [B + 1]); max_q is at least the largest number
of queries of a sequence.  Sequence b reads the prefix of its group and then its
lens[b] own tokens (int32 [B]), which lie on the pages pages[b] (int32 [B, W]) of
the caches (tilebench_amd.paged says how these are laid out; head dimension 64 or
128); its queries are its last tokens, each seeing the tokens up to its own.
Group g holds the sequences group_offsets[g] .. group_offsets[g + 1] - 1 (int32
[G + 1], from 0 to B); its prefix is prefix_lens[g] tokens (int32 [G]) on the pages
prefix_pages[g] (int32 [G, Wp]).  Without prefixes the three are None.  scale
defaults to D ** -0.5.  float8_e4m3fn caches come with k_scale and v_scale.  Rows
that see no token, and rows of no sequence, give 0 and -inf.

Lengths, offsets and page ids stay on the device and are clamped there.  No
counters, no state: the workspace is allocated per call.
"""
import ctypes
import functools

import torch

from tilebench_amd import paged
from tilebench_amd import runtime as rt

rt.load_library()

_last_config = None


@functools.lru_cache(maxsize=1024)
def workspace_bytes(*sizes) -> int:
    """Bytes of workspace of a call of these sizes (tb_shared_prefix_attention_workspace_size's, in its order)."""
    need = ctypes.c_int64(0)
    rt.call("tb_shared_prefix_attention_workspace_size", *sizes, ctypes.byref(need))
    return need.value


def check(q, k_cache, v_cache, prefix_pages, prefix_lens, group_offsets, pages, lens, cu_q, max_q, scale=None,
          k_scale=None, v_scale=None):
    """The sizes of a call; raises TypeError or ValueError for what run refuses (no GPU needed)."""
    op = "shared_prefix_attention"
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"{op}: q must be [tokens, heads, head_dim]")
    if q.dtype is not torch.float16 and q.dtype is not torch.bfloat16:
        raise TypeError(f"{op}: q must be float16 or bfloat16")
    T, Hq, D = shape
    Hkv = k_cache.shape[1] if k_cache.dim() == 4 else 0
    n_pages, page = paged.check_cache(op, q.dtype, Hkv, D, k_cache, v_cache, k_scale, v_scale)
    if D not in (64, 128) or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"{op}: need a head dimension of 64 or 128 and query heads that share the key/value heads "
                         f"(got {Hq} and {Hkv} heads of {D})")
    s_page, s_head, s_slot, _ = k_cache.stride()
    if (s_page | s_head | s_slot) * k_cache.element_size() % 16 or (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError(f"{op}: the caches' rows must be 16-byte aligned")
    if pages.dtype is not torch.int32 or lens.dtype is not torch.int32 or cu_q.dtype is not torch.int32:
        raise TypeError(f"{op}: page tables, lengths and offsets must be int32")
    table = pages.shape
    if len(table) != 2 or lens.shape != table[:1] or cu_q.dim() != 1 or cu_q.shape[0] != table[0] + 1:
        raise ValueError(f"{op}: pages must be [sequences, pages], lens [sequences], cu_q [sequences + 1]")
    B, W = table
    G = Wp = 0
    if prefix_pages is not None and prefix_lens is not None and group_offsets is not None:
        if prefix_pages.dtype is not torch.int32 or prefix_lens.dtype is not torch.int32 \
                or group_offsets.dtype is not torch.int32:
            raise TypeError(f"{op}: page tables, lengths and offsets must be int32")
        table = prefix_pages.shape
        if len(table) != 2 or prefix_lens.shape != table[:1] or group_offsets.dim() != 1 \
                or group_offsets.shape[0] != table[0] + 1:
            raise ValueError(f"{op}: prefix_pages must be [groups, pages], prefix_lens [groups], group_offsets "
                             "[groups + 1]")
        G, Wp = table
    elif prefix_pages is not None or prefix_lens is not None or group_offsets is not None:
        raise ValueError(f"{op}: prefix_pages, prefix_lens and group_offsets come together")
    if (G == 0) != (Wp == 0) or (T > 0 and (B < 1 or W < 1)):
        raise ValueError(f"{op}: empty page tables")
    if max_q < 0:
        raise ValueError(f"{op}: max_q must not be negative")
    return T, Hq, Hkv, D, G, Wp, B, W, n_pages, page


def run(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_pages, prefix_lens, group_offsets,
        pages: torch.Tensor, lens: torch.Tensor, cu_q: torch.Tensor, max_q: int, scale=None, k_scale=None,
        v_scale=None, **kwargs):
    global _last_config
    rt.require_device(q, k_cache, v_cache, prefix_pages, prefix_lens, group_offsets, pages, lens, cu_q, k_scale,
                      v_scale)
    T, Hq, Hkv, D, G, Wp, B, W, n_pages, page = check(q, k_cache, v_cache, prefix_pages, prefix_lens, group_offsets,
                                                      pages, lens, cu_q, max_q, scale, k_scale, v_scale)
    q = paged.aligned_rows(q, 8)
    q_st, q_sh, _ = q.stride()
    pages, lens, cu_q = pages.contiguous(), lens.contiguous(), cu_q.contiguous()
    if G:
        prefix_pages, prefix_lens = prefix_pages.contiguous(), prefix_lens.contiguous()
        group_offsets = group_offsets.contiguous()
    else:
        prefix_pages = prefix_lens = group_offsets = None
    out = paged.dense(q)
    lse = q.new_empty((T, Hq), dtype=torch.float32)
    cache_dtype = paged.DTYPES[k_cache.dtype]
    need = workspace_bytes(T, Hq, Hkv, D, G, Wp, B, W, page, max_q, cache_dtype)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    cs = k_cache.stride()
    ss = (0, 0, 0) if k_scale is None else k_scale.stride()
    rt.call("tb_shared_prefix_attention", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), rt.ptr(k_scale),
            rt.ptr(v_scale), rt.ptr(prefix_pages), rt.ptr(prefix_lens), rt.ptr(group_offsets), pages.data_ptr(),
            lens.data_ptr(), cu_q.data_ptr(), out.data_ptr(), lse.data_ptr(), T, Hq, Hkv, D, G, Wp, B, W, max_q,
            n_pages, page, q_st, q_sh, cs[0], cs[1], cs[2], *ss, D ** -0.5 if scale is None else scale,
            paged.DTYPES[q.dtype], cache_dtype, rt.ptr(ws), need, rt.stream_handle(q.get_device()))
    _last_config = {"kernels": ["attend", "combine"] if need else ["attend_each"], "workspace_bytes": need}
    return (out, lse)


def get_last_config():
    return _last_config
