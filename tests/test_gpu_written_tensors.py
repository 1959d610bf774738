"""Tensors that the operators write into on the caller's behalf (caches, q_out, out, lse) count as
written: a backward that saved their old values raises instead of computing with the new ones."""
import pytest
import torch

from inkling_fa4 import (_ops, inkling_fa4_rel_attention_decode_shared_prefix, inkling_kv_append,
                         inkling_qk_norm_rope)

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["ops", "ctypes"])
def path(request):
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = request.param
    yield
    _ops.USE_TORCH_OPS = before


def _randn(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _append(q=None, q_out=None, caches=None):
    """Four tokens of one sequence into the last of two pages."""
    caches = caches or [torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
                        for _ in range(2)]
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    table = torch.ones(1, 1, dtype=torch.int32, device="cuda")
    got = inkling_kv_append(_randn(4, 2, 128), _randn(4, 2, 128), *caches, table, cu, cu, q=q,
                            q_out=q_out)
    return got, caches


def test_caches(path):
    for q in (None, _randn(4, 2, 128)):
        _, caches = _append(q)
        assert [c._version for c in caches] == [1, 1]  # one write: zeros() made version 0


def test_queries_in_place(path):
    q = _randn(4, 2, 128)
    leaf = q.clone().requires_grad_()
    x = leaf * 1.0                             # not a leaf: written in place below
    y = inkling_qk_norm_rope(x, x.detach().clone())[0]  # saves x
    assert _append(x, q_out=x)[0] is x
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    q2 = leaf * 1.0
    y = inkling_qk_norm_rope(q2, q)[0]
    got, _ = _append(q2)                       # a new tensor for the queries: q2 is as it was
    assert not got.requires_grad and got.grad_fn is None
    y.sum().backward()


def test_inference_tensors(path):
    with torch.inference_mode():
        q = _randn(4, 2, 128)
        got, caches = _append(q, q_out=q)
        assert got is q and caches[0].is_inference()
    for q in (None, _randn(4, 2, 128)):        # tensors of inference mode outside of it
        _append(q, None, caches)


def test_shared_prefix_outputs(path):
    kc, vc = _randn(4, 16, 2, 128), _randn(4, 16, 2, 128)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1, 2], [0, 1, 3]], dtype=torch.int32, device="cuda")
    q, rel = _randn(2, 4, 128), _randn(2, 4, 16)
    out, lse = torch.empty_like(q), torch.empty(4, 2, device="cuda")
    inkling_fa4_rel_attention_decode_shared_prefix(q, kc, vc, rel, cu, cu * 40, 1, 40, 16, 32,
                                                   block_table=table, out=out, lse=lse)
    assert out._version == 1 and lse._version == 1
    assert kc._version == 0 and q._version == 0
