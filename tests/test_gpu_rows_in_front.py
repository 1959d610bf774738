"""Offsets that begin behind 0: the rows in front of the first sequence belong to none, as those behind
the last do."""
import numpy as np
import pytest
import torch

from inkling_fa4 import (_ops, inkling_fa4_rel_attention_decode_pages, inkling_kv_page_bounds,
                         inkling_kv_page_scores)
from long_context_cases import Case, np_
from oracle import long_context_oracle as oracle
from test_gpu_page_sparse import _check_scores

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("front", [1, 5, 40])
def test_scores_and_attention(front, path):
    c = Case([1, 3], [200, 90], 8, 2, 16, 50, seed=41, padding=front + 2)
    c.cu_q = c.cu_q + front
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    args = (c.q, bounds, c.rel, c.cu_q, c.cu_k, 3, 50, 16)
    kw = dict(block_table=c.table, softmax_scale=c.scale)
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        for _ in range(3):  # the memory that the new tensor gets
            torch.full((c.total, 2, c.width), 7.0, device="cuda")
        got = inkling_kv_page_scores(*args, **kw)
        given = torch.full((c.total, 2, c.width), 3.0, device="cuda")
        inkling_kv_page_scores(*args, out=given, **kw)
        out = inkling_fa4_rel_attention_decode_pages(
            c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 3, 200, 50,
            torch.zeros(c.total, 2, 1, dtype=torch.int32, device="cuda"), **kw)
    finally:
        _ops.USE_TORCH_OPS = before
    want, size = oracle.page_scores(np_(c.q), np_(bounds), np_(c.rel), np_(c.cu_q), np_(c.cu_k),
                                    np_(c.table), 16, 50, -1, c.scale)
    assert np.isneginf(want[:front]).all()
    _check_scores(got, want, size)
    assert torch.all(given[:front] == 3.0) and torch.all(given[front + 4:] == 3.0)
    assert torch.equal(given[front:front + 4], got[front:front + 4])
    assert not out[:front].any() and not out[front + 4:].any() and out[front:front + 4].any()
