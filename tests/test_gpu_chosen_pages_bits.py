"""Attention over chosen pages against the formula in 64 bits: the only rounding to 16 bits is the
output's.  The weights are two bf16 numbers each (2^-15 of their size is lost), everything else is held
in 32 bits."""
import numpy as np
import pytest
import torch

from inkling_fa4 import inkling_fa4_rel_attention_decode_pages
from long_context_cases import BF16, EPS32, Case, np_
from oracle import long_context_oracle as oracle
from test_gpu_page_sparse import choose

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(8, 2), (12, 4), (32, 1), (2, 2)])
@pytest.mark.parametrize("splits", [0, 1, 5, 11])
@pytest.mark.parametrize("page_size,window", [(16, -1), (64, 300)])
def test_only_the_output_is_rounded(page_size, window, splits, heads):
    c = Case([1, 1, 3], [900, 33, 470], *heads, page_size, 128, seed=21)
    pages = choose(c, 640 // page_size, window=window)
    want, weight, _, size = oracle.decode_pages(
        np_(c.q), np_(c.k), np_(c.v), np_(c.rel), np_(c.cu_q), np_(c.cu_k), np_(c.table), np_(pages),
        c.rel_extent, window, c.scale)
    got = np_(inkling_fa4_rel_attention_decode_pages(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, pages, (window, 0),
        block_table=c.table, softmax_scale=c.scale, num_splits=splits))
    # logits: 128 products and three more roundings of a step each (the matrix unit may cut off), and
    # 2^-21 of their size for the exponentials and their base
    logit = (131 * 2 * EPS32 + 2.0 ** -21) * size[..., None]
    # weights: the rest of a weight, at most 2^-7 of it, is rounded to 8 bits, which loses 2^-15 (2^-14
    # with the rest's own 2^-23); sums: two steps for each of up to 640 keys in two halves, the
    # factors of a tile and of the merges (64 more)
    tol = weight * (2 * logit + 2.0 ** -14 + (2 * 640 + 64) * 2 * EPS32)
    tol = tol * (1 + BF16) + BF16 * np.abs(want) + 1e-30
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("splits", [1, 3])
def test_infinite_values(splits):
    """An infinite value makes its column infinite, whatever the weight of its key: one that is a bf16
    number (the largest score's), or one with a rest."""
    c = Case([1, 1], [300, 200], 8, 2, 16, 30, seed=22)
    c.q[0] = 0.0
    c.rel[0] = 0.0  # all weights of the first row are 1
    pages = torch.arange(12, dtype=torch.int32, device="cuda").expand(2, 2, 12)
    for b in range(2):
        for i, key in enumerate((0, 5, 77, 130, 191)):
            c.v[c.table[b, key // 16].long(), key % 16, :, 3 * i] = float("inf" if i % 2 else "-inf")
    got = np_(inkling_fa4_rel_attention_decode_pages(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, 300, 30, pages, block_table=c.table,
        softmax_scale=c.scale, num_splits=splits))
    want = oracle.decode_pages(np_(c.q), np_(c.k), np_(c.v), np_(c.rel), np_(c.cu_q), np_(c.cu_k),
                               np_(c.table), np_(pages), 30, -1, c.scale)[0]
    odd = ~np.isfinite(want)
    assert odd.sum() == 2 * 8 * 5
    np.testing.assert_array_equal(got[odd], want[odd])
    assert np.isfinite(got[~odd]).all()
