"""Gathered weight into a buffer of any width through the C ABI, without accumulation: every place is
written, whatever the width, the window and the kernel that the call takes; nothing behind it is."""
import numpy as np
import pytest
import torch

from inkling_fa4 import _lib, _paged
from long_context_cases import EPS32, Case, np_
from oracle import long_context_oracle as oracle
from test_gpu_kv_evict import _lse

pytestmark = pytest.mark.gpu


def launch_mass(c, lse, mass, window, accumulate, max_q):
    p = _lib.AttentionMassParams()
    _paged.fill_seqs(p, c.cu_q, c.cu_k, c.table, c.page_size, c.pages)
    p.q, p.k_cache, p.rel = c.q.data_ptr(), c.k.data_ptr(), c.rel.data_ptr()
    p.lse, p.mass = lse.data_ptr(), mass.data_ptr()
    _paged.fill_strides(p, q=(c.q, ("t", "h")), k=(c.k, ("page", "t", "h")), rel=(c.rel, ("t", "h")),
                        lse=(lse, ("h", "t")), mass=(mass, ("b", "h")))
    p.total_q, p.n_heads, p.kv_heads, p.head_dim = c.total, c.heads, c.kv_heads, 128
    p.dtype, p.rel_extent, p.softmax_scale = _lib.IFA4_DTYPE_BF16, c.rel_extent, c.scale
    p.window_left, p.max_seqlen_q, p.max_seqlen_k = window, max_q, c.max_k
    p.mass_width, p.accumulate = mass.shape[2], accumulate
    _paged.launch("attention_mass", p, c.q.device)


@pytest.mark.parametrize("n_q,hint", [([1, 1, 1], 1), ([2, 0, 4], 4), ([5, 1, 40], 40), ([5, 1, 40], 1),
                                      ([90, 3, 130], 130)])
@pytest.mark.parametrize("window", [0, 35, 100, 336, -1])
@pytest.mark.parametrize("width", [1, 17, 20, 64, 250, 350, 400])
def test_every_place_is_written(width, window, n_q, hint):
    c = Case(n_q, [60, 352, 351], 8, 2, 16, 30, seed=1, padding=1)
    lse = _lse(c, window)
    want, err = oracle.attention_mass(np.zeros((3, 2, width)), np_(c.q), np_(c.k), np_(c.rel), np_(lse),
                                      np_(c.cu_q), np_(c.cu_k), np_(c.table), c.rel_extent, window,
                                      c.scale)
    wide = torch.full((3, 2, width + 40), float("nan"), device="cuda")
    launch_mass(c, lse, wide[:, :, :width], window, 0, hint)
    got = np_(wide)
    assert np.isnan(got[:, :, width:]).all()
    got = got[:, :, :width]
    # exponents: 128 products and four more roundings of a step each of the sizes they add up from;
    # exponentials: 2^-21 for theirs; sums: a rounding for every row and head, and one for the result
    tol = 132 * 2 * EPS32 * err + (2.0 ** -21 + (4 * max(n_q) + 3) * EPS32) * want
    assert np.array_equal(got[want == 0], want[want == 0])
    assert np.all(np.abs(got - want) <= tol + 1e-37)
