"""Bytes that the serving operators' configs count, against the sizes of generated tensors."""
import pytest
import torch
import yaml

from tilebench_amd.core.dtypes import resolve_dtype
from tilebench_amd.core.metrics import work
from tilebench_amd.data import tensors as T
from tilebench_amd.paths import operator_config


def _bytes(*tensors):
    return sum(t.numel() * t.element_size() for t in tensors)


def _work(op, case, dtype):
    return work(yaml.safe_load(open(operator_config(op)))["metrics"], case, dtype)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_an_append_reads_its_inputs_and_writes_its_rows(cache, dtype):
    case = dict(T=6, Hq=4, Hkv=2, D=64, page=4, axes=1, cache=cache)
    q, k, v, _, _, _, _, *pools = T.generate_rope_kv_append_inputs(**case, dtype=resolve_dtype(dtype), device="cpu")
    rows = pools[0].shape[0] * pools[0].shape[2]
    assert len(pools) == (4 if cache == "e4m3" else 2)
    assert _work("rope_kv_append", case, dtype)[1] == _bytes(q, k, v, q) + _bytes(*pools) / rows * 6


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_reads_every_token_once(cache, dtype):
    case = dict(B=4, prefix=32, own=16, n_q=2, Hq=4, Hkv=2, D=64, page=16, cache=cache)
    x = T.generate_shared_prefix_attention_inputs(**case, dtype=resolve_dtype(dtype), device="cpu")
    pools = [x[1], x[2], *x[11:]]
    slots = pools[0].shape[0] * pools[0].shape[2]
    tokens = 32 + 4 * 16 * 3 // 4            # sequences hold own / 2 to own tokens, three quarters on average
    assert _work("shared_prefix_attention", case, dtype)[1] == _bytes(*pools) / slots * tokens + 2 * _bytes(x[0])


def test_other_configs_are_counted_as_before():
    q, k = torch.zeros(8, 4, 64).half(), torch.zeros(8, 2, 64).half()
    assert _work("rotary_axes", dict(T=8, Hq=4, Hk=2, D=64, axes=1), "fp16")[1] == 2 * _bytes(q, k) + 4 * 8 + 4 * 64
