"""Sparse attention over pages against the oracle in 64 bits: bounds, scores, choice and attention, at
the lengths, groups, pages and masks where they can go wrong."""
import numpy as np
import pytest
import torch

from inkling_fa4 import (inkling_fa4_rel_attention_decode_pages, inkling_fa4_rel_attention_triton,
                         inkling_kv_page_bounds, inkling_kv_page_scores, inkling_kv_select_pages)
from long_context_cases import BF16, EPS32, SHAPES, Case, np_
from oracle import long_context_oracle as oracle

pytestmark = pytest.mark.gpu

# (query counts, key counts): single tokens, a chunk, empty sequences, more queries than keys
LENGTHS = [([1], [1]), ([1, 1, 1], [17, 300, 64]), ([3, 0, 1, 40], [50, 20, 0, 257]),
           ([5, 130], [3, 130])]


def _same(got, want):
    np.testing.assert_array_equal(np.asarray(got), np.asarray(want))


# --- bounds -----------------------------------------------------------------------------------

@pytest.mark.parametrize("heads", SHAPES)
@pytest.mark.parametrize("page_size", [16, 64, 256])
@pytest.mark.parametrize("n_q,n_k", LENGTHS)
def test_bounds(n_q, n_k, page_size, heads):
    c = Case(n_q, n_k, *heads, page_size, 8)
    bounds = torch.full((c.pages, c.kv_heads, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    want = oracle.page_bounds(np_(bounds), np_(c.k), np_(c.table), np_(c.cu_q), np_(c.cu_k))
    got = inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k, c.max_q, bounds=bounds)
    assert got is bounds
    _same(np_(got), want)


def test_bounds_of_all_pages_into_a_new_tensor_and_without_a_hint():
    c = Case([1, 2], [100, 700], 8, 2, 32, 8)
    want = oracle.page_bounds(np.zeros((c.pages, 2, 2, 128)), np_(c.k), np_(c.table), np_(c.cu_k),
                              np_(c.cu_k))
    _same(np_(inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)), want)
    _same(np_(inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k, 1)), want)  # a hint too small


def test_bounds_of_infinite_and_nan_keys_and_of_bad_pages():
    c = Case([90], [90], 4, 2, 16, 8)
    first = int(c.table[0, 0])
    c.k[first, 3, 0, 5] = float("inf")
    c.k[first, 4, 1, 6] = float("-inf")
    c.k[first, 7, 1, 9] = float("nan")
    c.table[0, 2], c.table[0, 3] = c.pages, -5  # no pages: nothing is written for them
    bounds = torch.zeros(c.pages, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    want = oracle.page_bounds(np_(bounds), np_(c.k), np_(c.table), np_(c.cu_q), np_(c.cu_k))
    _same(np_(inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k, 90, bounds=bounds)), want)
    assert np.isnan(want).any() and np.isinf(want).any()


# --- scores -----------------------------------------------------------------------------------

def _check_scores(got, want, size):
    """256 products (exact in fp32) are added up and scaled, then the bias is added: 260 roundings of
    at most a step (the matrix unit may cut off) of what the sizes of the terms add up to."""
    got = np_(got)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine])
    assert np.all(np.abs(got[fine] - want[fine]) <= 260 * 2 * EPS32 * size[fine])


def _scores(c, bounds, window=-1, first=0, last=0, **kw):
    want, size = oracle.page_scores(np_(c.q), np_(bounds), np_(c.rel), np_(c.cu_q), np_(c.cu_k),
                                    np_(c.table), c.page_size, c.rel_extent, window, c.scale, first,
                                    last)
    got = inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, c.max_q, c.rel_extent,
                                 c.page_size, (window, 0), block_table=c.table, softmax_scale=c.scale,
                                 first_pages=first, last_pages=last, **kw)
    return got, want, size


@pytest.mark.parametrize("heads", SHAPES + [(32, 1), (40, 2)])
@pytest.mark.parametrize("page_size,extent,window", [(16, 100, -1), (16, 7, 60), (64, 300, -1),
                                                     (256, 33, 200)])
@pytest.mark.parametrize("n_q,n_k", LENGTHS)
def test_scores(n_q, n_k, page_size, extent, window, heads):
    c = Case(n_q, n_k, *heads, page_size, extent, seed=1, padding=2)
    bounds = torch.zeros(c.pages, c.kv_heads, 2, 128, dtype=torch.bfloat16, device="cuda")
    inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k, bounds=bounds)
    got, want, size = _scores(c, bounds, window)
    _check_scores(got, want, size)


def test_scores_bound_every_logit():
    c = Case([1, 4], [200, 333], 8, 2, 16, 64, seed=2)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    got = np_(_scores(c, bounds)[0])
    q, rel = np_(c.q), np_(c.rel)
    for t in range(c.total):
        b, p = oracle.row_place(np_(c.cu_q), np_(c.cu_k), t)
        for h in range(8):
            k = oracle._rows(np_(c.k), np_(c.table)[b], np.arange(p + 1), h // 4)
            x = k @ q[t, h] * c.scale
            near = min(p + 1, 64)
            x[p + 1 - near:] += rel[t, h, :near][::-1]
            for j in range(p + 1):
                assert got[t, h // 4, j // 16] >= x[j] - 1e-4


@pytest.mark.parametrize("window", [-1, 100])
def test_scores_of_pages_that_are_always_taken(window):
    c = Case([1, 2], [400, 70], 8, 2, 16, 64, seed=3)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    got, want, size = _scores(c, bounds, window, 1, 2)
    _check_scores(got, want, size)
    assert np.isposinf(want).any()


def test_scores_of_layouts():
    """Merged projections, a bias shared by the tokens, a table column subset, an output of the caller's
    whose padding rows stay, hints that are too small."""
    c = Case([1, 9], [100, 200], 12, 4, 32, 50, seed=4, padding=3, merged=True, rel_broadcast=True)
    wide = torch.zeros(c.pages, 4, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    bounds = wide[:, :, 1]  # every third
    inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k, bounds=bounds)
    assert not wide[:, :, 0].any() and not wide[:, :, 2].any()
    out = torch.full((c.total, 4, c.width + 5), 3.0, device="cuda")[:, :, :c.width]
    c.max_q = 1
    got, want, size = _scores(c, bounds, out=out)
    assert got is out and torch.all(out[10:] == 3.0)
    _check_scores(got[:10], want[:10], size[:10])


def test_scores_of_nan_and_infinite_bounds():
    c = Case([1], [100], 4, 2, 16, 8, seed=5)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    bounds[c.table[0, 1], 0, 1, 3] = float("nan")
    bounds[c.table[0, 2], 1, 1, 3] = float("inf")
    c.table[0, 3] = -1  # no page: zeros
    q = np_(c.q)
    with np.errstate(invalid="ignore"):
        got, want, size = _scores(c, bounds)
    assert np.isnan(np_(got)[0, 0, 1])
    _check_scores(got, want, size)


# --- choice -----------------------------------------------------------------------------------

def _select(x, count, **kw):
    want = np.full(x.shape[:2] + (count,), -1, np.int32)
    host = x.cpu().numpy()
    for t in range(x.shape[0]):
        for g in range(x.shape[1]):
            at = oracle.select_largest(host[t, g], count)
            want[t, g, :len(at)] = at
    _same(np_(inkling_kv_select_pages(x, count, **kw)), want)


@pytest.mark.parametrize("width,count", [(1, 1), (1, 5), (7, 3), (33, 33), (300, 40), (2048, 64),
                                         (2049, 1), (4097, 500), (5000, 4999), (20000, 1024)])
def test_select(width, count):
    g = torch.Generator().manual_seed(width)
    _select(torch.randn(3, 2, width, generator=g).cuda(), count)


def test_select_many_rows():
    g = torch.Generator().manual_seed(9)
    _select(torch.randn(300, 3, 50, generator=g).cuda(), 7)


@pytest.mark.parametrize("width", [100, 5000])
def test_select_ties_zeros_infinities_and_nan(width):
    g = torch.Generator().manual_seed(1)
    few = torch.randint(0, 4, (4, 2, width), generator=g).float() - 1.0
    few[few == 0] *= torch.where(torch.rand(int((few == 0).sum()), generator=g) < 0.5, -1.0, 1.0)
    for count in (1, width // 7, width // 2, width - 1, width + 3):
        _select(few.cuda(), count)
    odd = few.clone()
    odd[0, :, 3::7] = float("-inf")
    odd[1, :, 5::11] = float("nan")
    odd[2, :, 2::5] = float("inf")
    odd[3] = float("-inf")
    for count in (1, 20, width // 3, width):
        _select(odd.cuda(), count)
    # denormals, the largest and the smallest values, equal in all high bits
    x = torch.tensor([1e-45, -1e-45, 0.0, -0.0, 3.4e38, -3.4e38, 1.0, 1.0000001, 0.99999994, 1.0])
    _select(x.repeat(2, 1, 7).cuda(), 20)


def test_select_layouts():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 3, 130, generator=g).cuda()
    _select(x[:, :, 1:98], 10)           # rows that start between 16-byte boundaries
    _select(x[:1].expand(5, 3, 130), 10)  # one row for all
    _select(x.transpose(0, 1), 10)
    _select(x[:, :, ::2], 10)            # copied
    out = torch.full((5, 3, 20), 9, dtype=torch.int32, device="cuda")
    _select(x, 10, out=out[:, :, :10])
    assert torch.all(out[:, :, 10:] == 9)
    assert inkling_kv_select_pages(x[:0], 4).shape == (0, 3, 4)
    assert torch.all(inkling_kv_select_pages(x[:, :, :0], 4) == -1)


# --- attention --------------------------------------------------------------------------------

def choose(c, count, seed=0, window=-1):
    """Random choices of each row's pages, in random order, some entries no pages."""
    rng = np.random.default_rng(seed)
    pages = np.full((c.total, c.kv_heads, count), -1, np.int32)
    for t in range(c.total):
        at = oracle.row_place(np_(c.cu_q), np_(c.cu_k), t)
        if at is None or at[1] < 0:
            continue
        able = np.arange(at[1] // c.page_size + 1)
        for g in range(c.kv_heads):
            some = rng.permutation(able)[:max(1, rng.integers(0, count + 1))]
            pages[t, g, rng.permutation(count)[:len(some)]] = some[:count]
    return torch.from_numpy(pages).cuda()


def check_attention(c, pages, window=-1, got=None, lse=None, rows=None, **kw):
    want, weight, want_lse, size = oracle.decode_pages(
        np_(c.q), np_(c.k), np_(c.v), np_(c.rel), np_(c.cu_q), np_(c.cu_k), np_(c.table), np_(pages),
        c.rel_extent, window, c.scale)
    if got is None:
        got, lse = inkling_fa4_rel_attention_decode_pages(
            c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, pages, (window, 0),
            block_table=c.table, softmax_scale=c.scale, return_lse=True, **kw)
    got = np_(got)
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(got[odd], want[odd])
    got, want = np.where(odd, 0.0, got), np.where(odd, 0.0, want)
    # logits: 128 products and three more roundings of a step each, and 2^-21 of their size for the
    # exponentials and their base; weights: one rounding to bf16 each; output: one
    logit = (131 * 2 * EPS32 + 2.0 ** -21) * size[..., None]
    tol = weight * (BF16 + 2 * logit) * (1 + BF16) + BF16 * np.abs(want) * (1 + 2 * BF16) + 1e-30
    assert np.all((np.abs(got - want) <= tol) | odd), np.nanmax(np.abs(got - want) / tol)
    if lse is not None:
        fine = np.isfinite(want_lse)
        np.testing.assert_array_equal(np_(lse)[~fine], want_lse[~fine])
        err = np.abs(np_(lse)[fine] - want_lse[fine])
        assert np.all(err <= (logit[..., 0].T + 2.0 ** -20 * (1 + np.abs(want_lse)))[fine])


@pytest.mark.parametrize("heads", SHAPES + [(32, 1), (40, 2)])
@pytest.mark.parametrize("page_size,extent,window", [(16, 100, -1), (16, 7, 60), (64, 300, -1),
                                                     (256, 33, 200)])
@pytest.mark.parametrize("n_q,n_k", LENGTHS)
def test_attention(n_q, n_k, page_size, extent, window, heads):
    c = Case(n_q, n_k, *heads, page_size, extent, seed=6, padding=2)
    check_attention(c, choose(c, 5), window)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_attention_in_splits(splits):
    c = Case([1, 1, 3], [900, 33, 470], 8, 2, 16, 128, seed=7, padding=1)
    check_attention(c, choose(c, 41), num_splits=splits)


def test_attention_over_all_pages_is_the_attention():
    c = Case([1, 6], [500, 260], 8, 2, 32, 128, seed=8)
    pages = torch.arange(c.width, dtype=torch.int32, device="cuda").expand(c.total, 2, c.width)
    got = inkling_fa4_rel_attention_decode_pages(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, pages,
        block_table=c.table, softmax_scale=c.scale)
    dense = inkling_fa4_rel_attention_triton(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent,
        causal_align="bottom_right", block_table=c.table, softmax_scale=c.scale)
    check_attention(c, pages, got=got)
    # the bound above for either of the two
    check_attention(c, pages, got=dense)


def test_attention_entries_that_are_no_pages_and_repeated_ones():
    c = Case([1, 1], [200, 90], 4, 2, 16, 64, seed=9)
    pages = torch.tensor([[[2, 2, -1, 40, 5], [-7, 2 ** 31 - 1, -2 ** 31, 12, 12]],
                          [[-1] * 5, [100, 6, 7, 8, 9]]], dtype=torch.int32, device="cuda")
    check_attention(c, pages)
    c.table[0, 5] = -1           # listed, but no page: zero keys and values
    c.table[0, 2] = c.pages + 3
    check_attention(c, pages)


def test_attention_of_nan_infinite_and_lowest_values():
    c = Case([1, 1, 1, 1], [100] * 4, 4, 2, 16, 64, seed=10)
    pages = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda").expand(4, 2, 3).contiguous()
    page = c.table[:, 2].long()
    c.k[page[0], 1, 0, 0] = float("nan")
    c.rel[1, 2, 70 - 64] = float("-inf")  # a key whose bias hides it
    c.rel[1, :2] = torch.finfo(torch.bfloat16).min
    c.k[page[2], 3, 1, 0] = float("inf")
    c.v[page[3], 3, 1, 0] = float("inf")
    c.v[c.table[3, 1].long()] = float("nan")  # not chosen
    c.q[2, :, 0] = c.q[2, :, 0].abs() + 1.0
    q = np_(c.q)
    check_attention(c, pages)


def test_attention_where_every_bias_hides():
    """All keys of a row hidden by -inf: 0 and lse -inf, alone and in splits."""
    c = Case([1], [60], 4, 2, 16, 64, seed=11)
    c.rel[:] = float("-inf")
    pages = torch.arange(4, dtype=torch.int32, device="cuda").expand(1, 2, 4)
    for splits in (1, 3):
        check_attention(c, pages, num_splits=splits)


@pytest.mark.parametrize("splits", [1, 2, 5])
def test_attention_where_every_bias_is_the_lowest(splits):
    """The mean of the values, whatever the split (the lse is out of range there)."""
    c = Case([1, 1], [60, 200], 4, 2, 16, 64, seed=11)
    c.rel[:] = torch.finfo(torch.bfloat16).min
    pages = torch.tensor([[0, 1, 2, 3, 12], [9, 10, 11, 12, 3]], dtype=torch.int32, device="cuda")
    pages = pages[:, None, :].expand(2, 2, 5).contiguous()
    pages[1, :, 4] = -1
    got = inkling_fa4_rel_attention_decode_pages(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, 200, 64, pages, block_table=c.table,
        softmax_scale=c.scale, num_splits=splits)
    check_attention(c, pages, got=got)


def test_attention_outputs_of_the_caller():
    c = Case([1, 2], [100, 200], 12, 4, 32, 50, seed=12, padding=3, merged=True, rel_broadcast=True)
    pages = choose(c, 4)
    for splits in (1, 3):
        wide = torch.full((c.total, 14, 128), 5.0, dtype=torch.bfloat16, device="cuda")
        out, lse = wide[:, 1:13], torch.full((12, c.total), 5.0, device="cuda")
        got = inkling_fa4_rel_attention_decode_pages(
            c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, pages,
            block_table=c.table, softmax_scale=c.scale, out=out, lse=lse, num_splits=splits)
        assert got[0] is out and got[1] is lse
        assert torch.all(wide[:, 0] == 5.0) and torch.all(wide[:, 13] == 5.0)
        assert torch.all(out[3:] == 5.0) and torch.all(lse[:, 3:] == 5.0)
        out[3:], lse[:, 3:] = 0.0, float("-inf")
        check_attention(c, pages, got=out, lse=lse)


def test_attention_strided_choice_and_empty_choice():
    c = Case([1, 1], [100, 200], 8, 2, 16, 50, seed=13)
    pages = choose(c, 6)
    check_attention(c, pages.repeat_interleave(2, dim=2)[:, :, ::2])
    check_attention(c, pages.transpose(0, 1).contiguous().transpose(0, 1))
    check_attention(c, pages[:, :, :0])
