"""The fresh-input checks of tilebench_amd.core.anticache on the serving operators:
fresh inputs, new values written in place into the same tensors, and a repeat,
each against the operator's torch reference.  Appends write their caches (and the
scales), which they return; nothing else is written."""
import importlib
import itertools

import pytest
import torch
import yaml

from tilebench_amd.core.anticache import CHECKS, numerical_checks
from tilebench_amd.core.verifier import config_tolerance
from tilebench_amd.data import tensors as T
from tilebench_amd.hardware import detect_arch
from tilebench_amd.paths import list_serving_operators, operator_config

pytestmark = pytest.mark.gpu

CASES = [
    ("rotary_axes", dict(T=130, axes=3, Hq=6, Hk=2, D=96), torch.float16, ()),
    ("rotary_axes", dict(T=33, axes=1, Hq=4, Hk=4, D=64), torch.float32, ()),
    ("rope_kv_append", dict(T=64, axes=2, Hq=8, Hkv=2, D=64, page=16, cache="same"), torch.bfloat16, (7, 8)),
    ("rope_kv_append", dict(T=64, axes=1, Hq=8, Hkv=2, D=128, page=16, cache="e4m3"), torch.float16, (7, 8, 9, 10)),
    ("shared_prefix_attention", dict(B=9, prefix=130, own=70), torch.float16, ()),
    ("shared_prefix_attention", dict(B=9, prefix=1300, own=200), torch.bfloat16, ()),
]


def test_every_serving_operator_has_a_case():
    assert {op for op, *_ in CASES} == set(list_serving_operators())


@pytest.mark.parametrize("op,case,dtype,mutable", CASES, ids=[f"{op}-{i}" for i, (op, *_) in enumerate(CASES)])
def test_fresh_inputs_same_address_and_repeat(gpu, op, case, dtype, mutable):
    print("[gpu case] anticache", op, case, dtype, flush=True)
    impl_hip = importlib.import_module(f"tilebench_amd.benchmarks.serving.{op}.impl_hip")
    impl_torch = importlib.import_module(f"tilebench_amd.benchmarks.serving.{op}.impl_torch")
    atol, rtol = config_tolerance(yaml.safe_load(open(operator_config(op)))["verify"], detect_arch())
    seeds = itertools.count(50)

    def make():
        x = T.get_generator(op)(**case, dtype=dtype, seed=next(seeds), device="cpu")
        return tuple(t.to("cuda") if isinstance(t, torch.Tensor) else t for t in x)

    res = numerical_checks(impl_hip.run, impl_torch.run, make, atol=atol, rtol=rtol, mutable=mutable,
                           allow_aliasing=bool(mutable))
    assert [r.name for r in res] == list(CHECKS), res[-1].message
    assert all(r.ok for r in res), [r.message for r in res if not r.ok]
    for r in res:
        assert set(r.aliased_inputs) == set(mutable) and set(r.mutated_inputs) <= set(mutable)
