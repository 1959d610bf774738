"""Tracers do not see the operators next to the attention (they are no dispatcher operators): a traced
call is refused, where it would become a constant of the graph and the append's writes would be lost.
Modes that only look on leave the results as they are."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from inkling_fa4 import (_ops, inkling_bucket_bias, inkling_bucket_bias_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix, inkling_kv_append,
                         inkling_qk_norm_rope, inkling_qk_norm_rope_backward)

pytestmark = pytest.mark.gpu


def _randn(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _calls():
    x, kc, vc = _randn(4, 2, 128), _randn(3, 16, 2, 128), _randn(3, 16, 2, 128)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    one = torch.arange(5, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    pages = torch.tensor([[1, 2]] * 4, dtype=torch.int32, device="cuda")
    rel, starts = _randn(4, 2, 16), torch.arange(8, dtype=torch.int32, device="cuda")
    weights = torch.randn(8, 2, device="cuda")
    return x, {
        "norm": lambda x: inkling_qk_norm_rope(x, x)[0],
        "norm_grad": lambda x: inkling_qk_norm_rope_backward(x, x, x, x)[0],
        "append": lambda x: inkling_kv_append(x, x, kc, vc, table, cu, cu, q=x),
        "append_keys": lambda x: [inkling_kv_append(x, x, kc, vc, table, cu, cu), kc.clone()][1],
        "prefix": lambda x: inkling_fa4_rel_attention_decode_shared_prefix(
            x, kc, vc, rel, one, one * 20, 1, 20, 16, 16, block_table=pages),
        "bias": lambda x: inkling_bucket_bias(weights, starts, 4, 16),
        "bias_grad": lambda x: inkling_bucket_bias_backward(rel, starts, 8)}


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("name", ["norm", "norm_grad", "append", "append_keys", "prefix", "bias",
                                  "bias_grad"])
def test_refused(name, path):
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        x, calls = _calls()
        f = calls[name]
        for traced in (lambda: make_fx(f)(x), lambda: torch.jit.trace(f, x)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                traced()
        f(x)  # and not afterwards
    finally:
        _ops.USE_TORCH_OPS = before


class _LooksOn(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_other_modes():
    x, calls = _calls()
    for f in calls.values():
        want = f(x)
        with _LooksOn():
            got = f(x)
        assert torch.equal(got, want)
