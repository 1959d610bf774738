"""Gathered attention weight and eviction against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from inkling_fa4 import (inkling_fa4_rel_attention_triton, inkling_kv_attention_mass, inkling_kv_evict)
from long_context_cases import EPS32, SHAPES, Case, np_
from oracle import long_context_oracle as oracle

pytestmark = pytest.mark.gpu

LENGTHS = [([1], [1]), ([1, 1, 1], [17, 600, 256]), ([3, 0, 1, 40], [50, 20, 0, 300]),
           ([5, 130], [3, 130])]


def _lse(c, window):
    return inkling_fa4_rel_attention_triton(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, True, (window, 0),
        causal_align="bottom_right", block_table=c.table, softmax_scale=c.scale, return_lse=True)[1]


def _check_mass(c, lse, window=-1, mass=None, **kw):
    width = c.width * c.page_size if mass is None else mass.shape[2]
    start = np.zeros((len(c.n_q), c.kv_heads, width)) if mass is None else np_(mass)
    want, err = oracle.attention_mass(start, np_(c.q), np_(c.k), np_(c.rel), np_(lse), np_(c.cu_q),
                                      np_(c.cu_k), np_(c.table), c.rel_extent, window, c.scale)
    got = inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, c.max_q, c.max_k,
                                    c.rel_extent, (window, 0), block_table=c.table,
                                    softmax_scale=c.scale, mass=mass, **kw)
    assert mass is None or got is mass
    odd = ~np.isfinite(want)
    got = np_(got)
    np.testing.assert_array_equal(got[odd], want[odd])
    got, want, err = (np.where(odd, 0.0, x) for x in (got, want, err))
    # exponents: 128 products and four more roundings of a step each of the sizes they add up from;
    # exponentials: 2^-21 for theirs; sums: a rounding for every row and head, and one for the result
    terms = max(c.n_q) * (c.heads // c.kv_heads) + 2
    tol = 132 * 2 * EPS32 * err + (2.0 ** -21 + terms * EPS32) * np.abs(want - start) + EPS32 * np.abs(want)
    assert np.all(np.abs(got - want) <= tol + 1e-37), np.max(np.abs(got - want) / (tol + 1e-37))


@pytest.mark.parametrize("heads", SHAPES + [(32, 1), (256, 2)])
@pytest.mark.parametrize("page_size,extent,window", [(16, 100, -1), (16, 7, 60), (64, 300, -1),
                                                     (256, 33, 200)])
@pytest.mark.parametrize("n_q,n_k", LENGTHS)
def test_mass(n_q, n_k, page_size, extent, window, heads):
    if heads[0] == 256 and (page_size != 16 or extent != 100):
        pytest.skip("one layout of the largest group")
    c = Case(n_q, n_k, *heads, page_size, extent, seed=1, padding=2)
    _check_mass(c, _lse(c, window), window)


def test_mass_of_a_prompt_over_many_tiles():
    c = Case([700, 90], [700, 600], 8, 2, 64, 130, seed=2)
    _check_mass(c, _lse(c, -1))
    _check_mass(c, _lse(c, 333), 333)


def test_mass_is_added_in_place_and_only_at_keys():
    c = Case([1, 4], [100, 300], 8, 2, 16, 64, seed=3)
    lse = _lse(c, -1)
    wide = torch.randn(2, 2, 400, device="cuda").abs()
    before = wide.clone()
    _check_mass(c, lse, mass=wide[:, :, :310])
    assert torch.equal(wide[:, :, 310:], before[:, :, 310:])
    assert torch.equal(wide[0, :, 100:], before[0, :, 100:])
    assert torch.equal(wide[1, :, 300:], before[1, :, 300:])
    _check_mass(c, lse, mass=wide[:, :, :250])  # keys without a place
    c.max_q = c.max_k = 1  # hints that are too small
    _check_mass(c, lse, mass=wide[:, :, :310])
    _check_mass(c, lse)


def test_mass_sums_to_the_number_of_heads():
    """Every query gives a weight of one per head: fp32 sums of 500 weights, each with an exponent off
    by at most 132 steps of the sizes it adds up from (under 64 here) and as much in lse."""
    c = Case([50], [500], 8, 2, 32, 64, seed=4)
    mass = inkling_kv_attention_mass(c.q, c.k, c.rel, _lse(c, -1), c.cu_q, c.cu_k, 50, 500, 64,
                                     block_table=c.table, softmax_scale=c.scale)
    np.testing.assert_allclose(np_(mass).sum(-1), 50 * 4, rtol=2 * 132 * 2 * EPS32 * 64)


def test_mass_of_layouts_rows_without_keys_and_nan():
    c = Case([3, 2], [100, 1], 12, 4, 32, 50, seed=5, padding=3, merged=True, rel_broadcast=True)
    lse = _lse(c, -1)
    assert torch.isneginf(lse[:, 3]).all()  # two queries of a sequence with one key
    wide = torch.full((c.total, 14), float("nan"), device="cuda")
    wide[:, 1:13] = lse.t()
    _check_mass(c, wide[:, 1:13].t())
    c.k[c.table[0, 1].long(), 3, 1, 0] = float("nan")
    c.k[c.table[0, 1].long(), 5, 2, 0] = float("-inf")
    _check_mass(c, lse)
    lse[2, 1] = float("nan")
    _check_mass(c, lse)
    c.table[0, 2] = -1  # no page: zero keys
    lse[2, 1] = 1.0
    _check_mass(c, lse)


def test_mass_is_the_same_every_time():
    c = Case([200, 1], [300, 1000], 8, 2, 16, 64, seed=6)
    lse = _lse(c, -1)
    a, b = (inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, 200, 1000, 64,
                                      block_table=c.table) for _ in range(2))
    assert torch.equal(a, b)


# --- eviction ---------------------------------------------------------------------------------

def _check_evict(c, mass, budget, first=0, recent=0):
    want = oracle.kv_evict(c.k.float().cpu().numpy(), c.v.float().cpu().numpy(), mass.cpu().numpy(),
                           np_(c.table), np_(c.cu_k), budget, first, recent)
    before = mass.clone()
    kept, left, cu = inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, budget, first=first,
                                      recent=recent)
    np.testing.assert_array_equal(kept.cpu().numpy(), want[2])
    np.testing.assert_array_equal(left.cpu().numpy(), want[3])
    np.testing.assert_array_equal(cu.cpu().numpy(), want[4])
    np.testing.assert_array_equal(c.k.float().cpu().numpy(), want[0])
    np.testing.assert_array_equal(c.v.float().cpu().numpy(), want[1])
    assert torch.equal(before.view(torch.int32), mass.view(torch.int32))


def _mass(c, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(len(c.n_k), c.kv_heads, c.width * c.page_size, generator=g) * 2).exp().cuda()


@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("page_size", [16, 64, 256])
@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (1, 0, 1), (64, 4, 20), (100, 100, 0),
                                                 (100, 0, 100), (250, 3, 100), (2000, 5, 9)])
def test_evict(budget, first, recent, page_size, heads):
    c = Case([1] * 5, [17, 600, 0, 64, 1100], *heads, page_size, 8, seed=1)
    _check_evict(c, _mass(c), budget, first, recent)


def test_evict_long():
    c = Case([1, 1], [9000, 5003], 4, 2, 64, 8, seed=2)
    _check_evict(c, _mass(c), 3001, 4, 128)


def test_evict_ties_infinities_and_nan():
    c = Case([1] * 3, [300, 280, 150], 8, 2, 16, 8, seed=3)
    mass = torch.randint(0, 3, (3, 2, c.width * 16), generator=torch.Generator().manual_seed(0))
    mass = mass.float().cuda()
    mass[0, 0, 5::9] = float("nan")
    mass[0, 1, 5::9] = float("inf")
    mass[1, 0, :250] = float("-inf")
    mass[1, 1] = float("-inf")
    mass[2] = 0.0
    _check_evict(c, mass, 100, 2, 30)


def test_evict_narrow_and_strided_masses():
    c = Case([1, 1], [300, 200], 4, 2, 16, 8, seed=4)
    mass = _mass(c)
    _check_evict(c, mass[:, :, :180], 60, 0, 10)  # keys without a mass
    c = Case([1, 1], [300, 200], 4, 2, 16, 8, seed=4)
    _check_evict(c, mass[:, :1].expand(2, 2, mass.shape[2]), 60, 1, 10)


def test_evict_places_without_pages():
    c = Case([1, 1], [300, 200], 4, 2, 16, 8, seed=5)
    c.table[0, 1], c.table[0, 17], c.table[1, 12] = -1, c.pages, -3
    _check_evict(c, _mass(c), 60, 0, 40)


def test_evict_twice_and_append_room():
    c = Case([1], [500], 8, 2, 16, 8, seed=6)
    mass = _mass(c)
    _check_evict(c, mass, 200, 4, 30)
    kept, left, c.cu_k = inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, 200, first=4, recent=30)
    assert int(c.cu_k[1]) == 200 and not left[:, :, 200:].any()
    _check_evict(c, left, 90, 4, 30)
