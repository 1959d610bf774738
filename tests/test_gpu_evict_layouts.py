"""Eviction from caches that are slices of one tensor, in every order, and from caches that share
elements, which is refused without a write."""
import numpy as np
import pytest
import torch

from inkling_fa4 import _lib, _ops, inkling_kv_evict
from long_context_cases import Case
from test_gpu_kv_evict import _check_evict, _mass

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["pkths", "ptkhs", "pthks", "kpths", "pkhts"])
def test_slices_of_one_tensor(order):
    """p pages, t tokens, h heads, s values; k: keys and values."""
    c = Case([1, 1], [300, 170], 8, 2, 16, 8, seed=61)
    both = torch.stack((c.k, c.v)).permute(*("kpths".index(x) for x in order)).contiguous()
    both = both.permute(*(order.index(x) for x in "kpths"))
    c.k, c.v = both[0], both[1]
    _check_evict(c, _mass(c), 70, 3, 20)


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
def test_caches_that_share_elements_are_refused(path):
    c = Case([1], [300], 8, 2, 16, 8, seed=62)
    pool = torch.randn(c.k.numel() + 4096, device="cuda").to(torch.bfloat16)
    c.k, c.v = pool[:c.k.numel()].view(c.k.shape), pool[4096:].view(c.k.shape)  # shifted by a page
    before, mass = pool.clone(), _mass(c)
    was = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        with pytest.raises(_lib.Ifa4Error, match="k_cache and v_cache share memory"):
            inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, 70)
    finally:
        _ops.USE_TORCH_OPS = was
    assert torch.equal(pool, before)
