"""Forward-mode differentiation of the differentiable entry points is refused: a dual tensor needs no
gradient, so a call that looked for one would return an output without the tangent.  The refusal comes
before any kernel: the entry points' autograd functions have no forward-mode formula."""
import pytest
import torch
from torch.autograd import forward_ad

from inkling_fa4 import _ops, bucket_bias, inkling_bucket_bias, inkling_qk_norm_rope, qk_norm_rope


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.fixture
def no_kernel(monkeypatch):
    """The forwards without a GPU: outputs of the right shapes."""
    monkeypatch.setattr(qk_norm_rope, "_forward", lambda q, k, *rest: (q.clone(), k.clone()))
    monkeypatch.setattr(bucket_bias, "_forward",
                        lambda table, starts, t, r: table.new_zeros(t, table.shape[1], r))


@pytest.mark.parametrize("which", range(4))
def test_norm_rope(no_kernel, which):
    x, w = torch.randn(3, 2, 128, dtype=torch.bfloat16), torch.ones(128)
    with forward_ad.dual_level():
        args = [x, x.clone(), w, w.clone()]
        args[which] = _dual(args[which])
        with pytest.raises(NotImplementedError, match="forward mode"):
            inkling_qk_norm_rope(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            inkling_qk_norm_rope(*args)
        out = inkling_qk_norm_rope(x, x, w, w)  # nothing dual: an ordinary call
        assert torch.equal(out[0], x) and not out[0].requires_grad


def test_bucket_bias(no_kernel):
    starts = torch.tensor([0, 1], dtype=torch.int32)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            inkling_bucket_bias(_dual(torch.ones(2, 4)), starts, 3, 8)
        assert inkling_bucket_bias(torch.ones(2, 4), starts, 3, 8).shape == (3, 4, 8)


def test_which_calls_go_through_the_autograd_function():
    x, leaf = torch.ones(2), torch.ones(2, requires_grad=True)
    assert not _ops.differentiates(x, None, "no tensor")
    assert _ops.differentiates(x, None, leaf)
    with torch.no_grad():
        assert not _ops.differentiates(leaf)
    with forward_ad.dual_level():
        assert _ops.differentiates(x)
    assert not _ops.differentiates(x)
