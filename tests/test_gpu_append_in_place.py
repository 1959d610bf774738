"""The append's queries in place: refused where k or v have elements in common with them (they would be
read while they are written), the same result as into a new tensor where they have none."""
import pytest
import torch

from inkling_fa4 import inkling_kv_append

pytestmark = pytest.mark.gpu


def _randn(*shape):
    return torch.randn(*shape, device="cuda").to(torch.bfloat16)


def _append(q, k, v, **kw):
    caches = [torch.zeros(1, 16, k.shape[1], 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cu = torch.tensor([0, k.shape[0]], dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    inv = (100.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).cuda()
    got = inkling_kv_append(k, v, *caches, table, cu, cu, q=q, inv_freq=inv, **kw)
    return got, *caches


def test_refused():
    x, y = _randn(5, 4, 128), _randn(5, 4, 128)
    before = x.clone()
    for q, k, v in ((x, x, y), (x, y, x), (x, x[:, 3:], y[:, 3:]), (x[:, :2], y[:, :2], x[:, 1:3])):
        with pytest.raises(ValueError, match="in common with q_out"):
            _append(q, k, v, q_out=q)
    assert torch.equal(x, before)
    got = _append(x, x, x)  # into a new tensor: nothing is written that is read
    assert torch.equal(got[2][0, :5], x) and torch.equal(got[0], got[1][0, :5])


@pytest.mark.parametrize("layout", ["merged", "turns", "stacked"])
def test_layouts_of_a_layer(layout):
    if layout == "merged":
        merged = _randn(7, 8 * 128)
        q, k, v = (merged[:, a * 128:b * 128].view(7, b - a, 128) for a, b in ((0, 4), (4, 6), (6, 8)))
    elif layout == "turns":
        q, k, v = _randn(7, 4, 3, 128).unbind(2)
    else:
        q, k, v = _randn(3, 7, 4, 128).unbind(0)
    kv = k.clone(), v.clone()
    want = _append(q, k, v)
    got = _append(q, k, v, q_out=q)
    assert got[0] is q and all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(kv[0], k) and torch.equal(kv[1], v)
