"""The long-context operators as they are used together, captured, side by side on streams, and at
sizes that the per-operator tests leave out.  Every stage is compared with the oracle on the inputs it
was given (the outputs of the stage before)."""
import math

import numpy as np
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import inkling_fa4
from inkling_fa4 import (_lib, _ops, inkling_fa4_rel_attention_decode_pages,
                         inkling_fa4_rel_attention_triton, inkling_kv_append,
                         inkling_kv_attention_mass, inkling_kv_evict, inkling_kv_page_bounds,
                         inkling_kv_page_scores, inkling_kv_select_pages)
from long_context_cases import BF16, EPS32, Case, cu, np_
from oracle import long_context_oracle as oracle
from test_gpu_kv_evict import _check_evict, _check_mass, _lse, _mass
from test_gpu_page_sparse import _check_scores, _select, check_attention, choose

pytestmark = pytest.mark.gpu


def _step(c, bounds, selected=6):
    """One decode step behind an append: bounds, scores, choice, attention."""
    inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k, c.max_q, bounds=bounds)
    scores = inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, c.max_q, c.rel_extent,
                                    c.page_size, block_table=c.table, softmax_scale=c.scale,
                                    first_pages=1, last_pages=2)
    pages = inkling_kv_select_pages(scores, selected)
    out = inkling_fa4_rel_attention_decode_pages(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent, pages,
        block_table=c.table, softmax_scale=c.scale)
    return scores, pages, out


def test_a_run_of_all():
    """Two sequences: append, sparse decode, gathered weights, eviction, and once more behind it."""
    extent, budget = 40, 96
    c = Case([1, 1], [300, 171], 8, 2, 16, extent, seed=1)
    gen = torch.Generator().manual_seed(2)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    mass = torch.zeros(2, 2, c.width * 16, device="cuda")
    for turn in range(3):
        # the new token (the case has it in place at first: written again from new values)
        new = [torch.randn(2, 2, 128, generator=gen).to(torch.bfloat16).cuda() for _ in range(2)]
        inkling_kv_append(*new, c.k, c.v, c.table, c.cu_q, c.cu_k, eps=None)
        for b, n in enumerate((c.cu_k[1:] - c.cu_k[:-1]).tolist()):
            at = c.table[b, (n - 1) // 16].long(), (n - 1) % 16
            assert torch.equal(c.k[at], new[0][b]) and torch.equal(c.v[at], new[1][b])
        want = oracle.page_bounds(np_(bounds), np_(c.k), np_(c.table), np_(c.cu_q), np_(c.cu_k))
        scores, pages, out = _step(c, bounds)
        np.testing.assert_array_equal(np_(bounds), want)
        _check_scores(scores, *oracle.page_scores(np_(c.q), want, np_(c.rel), np_(c.cu_q), np_(c.cu_k),
                                                  np_(c.table), 16, extent, -1, c.scale, 1, 2))
        host = np_(scores)
        for t in range(2):
            for g in range(2):
                at = oracle.select_largest(host[t, g], 6)
                np.testing.assert_array_equal(np_(pages)[t, g], at + [-1] * (6 - len(at)))
        check_attention(c, pages, got=out)
        _check_mass(c, _lse(c, -1), mass=mass)
        if turn == 1:
            before, length = (c.k.clone(), c.v.clone()), c.cu_k.clone()
            want = oracle.kv_evict(c.k.float().cpu().numpy(), c.v.float().cpu().numpy(),
                                   mass.cpu().numpy(), np_(c.table), np_(c.cu_k), budget, 2, extent)
            kept, mass, c.cu_k = inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, budget, first=2,
                                                  recent=extent)
            np.testing.assert_array_equal(kept.cpu().numpy(), want[2])
            np.testing.assert_array_equal(c.k.float().cpu().numpy(), want[0])
            np.testing.assert_array_equal(mass.cpu().numpy(), want[3])
            _attends_as_before(c, before, length, kept)
            inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k, bounds=bounds)
        # room for the next token
        c.cu_k = c.cu_k + torch.arange(3, dtype=torch.int32, device="cuda")
        c.max_k = int((c.cu_k[1:] - c.cu_k[:-1]).max())


def _attends_as_before(c, before, length, kept):
    """With recent >= rel_extent the attention over what is left is the attention over the kept keys
    at the places, and with the biases, they had."""
    out = inkling_fa4_rel_attention_triton(
        c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, c.max_k, c.rel_extent, causal_align="bottom_right",
        block_table=c.table, softmax_scale=c.scale)
    k, v = (np_(x) for x in before)
    q, rel, n_k = np_(c.q), np_(c.rel), np.diff(np_(length))
    for b in range(2):
        p = n_k[b] - 1
        for h in range(8):
            at = np_(kept)[b, h // 4]
            at = at[at >= 0]
            keys, values = (oracle._rows(x, np_(c.table)[b], at, h // 4) for x in (k, v))
            d = p - at
            x = keys @ q[b, h] * c.scale + np.where(d < c.rel_extent, rel[b, h][np.minimum(d, c.rel_extent)], 0)
            w = np.exp(x - x.max())
            want, size = w @ values / w.sum(), w @ np.abs(values) / w.sum()
            # P and the output rounded to bf16; the logits are good to 2^-12 at this size
            assert np.all(np.abs(np_(out)[b, h] - want) <= size * (BF16 + 2.0 ** -11) + BF16 * np.abs(want))


def test_captured_and_replayed_with_new_inputs():
    c = Case([1, 1, 1], [200, 33, 500], 8, 2, 16, 64, seed=3)
    bounds = torch.zeros(c.pages, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k, bounds=bounds)
    lse = _lse(c, -1)
    mass = torch.zeros(3, 2, c.width * 16, device="cuda")

    def run():
        outs = _step(c, bounds, 12)
        inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, 1, 500, 64, block_table=c.table,
                                  softmax_scale=c.scale, mass=mass)
        many = inkling_fa4_rel_attention_decode_pages(
            c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, 500, 64, outs[1], block_table=c.table,
            softmax_scale=c.scale, num_splits=11)
        return outs + (many, mass) + inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, 100, first=1,
                                                      recent=64)

    stream = torch.cuda.Stream()
    state = [t.clone() for t in (c.k, c.v, bounds)]

    def restore():
        for t, s in zip((c.k, c.v, bounds), state):
            t.copy_(s)
        mass.zero_()

    with torch.cuda.stream(stream):
        run()
        restore()
        graphs = []
        for _ in range(2):  # two of them, with workspaces of their own
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs = run()
            graphs.append((g, outs))
    torch.cuda.synchronize()
    for seed, (g, outs) in zip((7, 8, 9, 10), graphs * 2):
        restore()
        new = torch.randn(c.q.shape, generator=torch.Generator().manual_seed(seed))
        c.q.copy_(new.to(torch.bfloat16))
        lse.copy_(_lse(c, -1))
        c.cu_k.copy_(cu([180 + seed, 20 + seed, 490 + seed % 10]))
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs] + [c.k.clone(), c.v.clone()]
        restore()
        want = run()
        for a, b in zip(got, list(want) + [c.k, c.v]):
            assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a,
                               b.nan_to_num(7.0) if b.is_floating_point() else b)


def test_side_by_side_on_streams():
    cases = [Case([1, 2], [700 + 100 * i, 90], 8, 2, 16, 64, seed=20 + i) for i in range(4)]
    masses = [_mass(c, i) for i, c in enumerate(cases)]
    want = [oracle.kv_evict(c.k.float().cpu().numpy(), c.v.float().cpu().numpy(), m.cpu().numpy(),
                            np_(c.table), np_(c.cu_k), 200, 1, 64) for c, m in zip(cases, masses)]
    pages = [choose(c, 30) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for c, p, s in zip(cases, pages, streams):
        with torch.cuda.stream(s):
            outs.append([inkling_fa4_rel_attention_decode_pages(
                c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 2, 1000, 64, p, block_table=c.table,
                softmax_scale=c.scale, num_splits=n) for n in (1, 4, 12)])
    torch.cuda.synchronize()
    for c, p, o in zip(cases, pages, outs):
        for x in o:
            check_attention(c, p, got=x)
    got = []
    for c, m, s in zip(cases, masses, streams):
        with torch.cuda.stream(s):
            got.append(inkling_kv_evict(c.k, c.v, m, c.table, c.cu_k, 200, first=1, recent=64))
    torch.cuda.synchronize()
    for c, g, w in zip(cases, got, want):
        np.testing.assert_array_equal(g[0].cpu().numpy(), w[2])
        np.testing.assert_array_equal(c.k.float().cpu().numpy(), w[0])
        np.testing.assert_array_equal(c.v.float().cpu().numpy(), w[1])


def test_the_same_every_time():
    c = Case([1, 20], [900, 333], 12, 4, 16, 100, seed=4)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    first = _step(c, bounds, 20)
    for _ in range(20):
        for a, b in zip(first, _step(c, bounds, 20)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("width", [32769, 40001, 70000])
def test_select_rows_that_no_block_holds(width):
    g = torch.Generator().manual_seed(width)
    x = torch.randn(2, 1, width, generator=g).cuda()
    x[1] = x[1].round()  # many equal ones
    x[0, 0, 5] = float("nan")
    _select(x, 1000)
    _select(x, width - 3)


@pytest.mark.parametrize("width", [8193, 12345, 16384, 16385])
def test_select_wide_rows(width):
    g = torch.Generator().manual_seed(width)
    x = torch.randn(2, 2, width, generator=g).cuda()
    x[1] = x[1].round()
    for count in (1, 700, width - 1):
        _select(x, count)


@pytest.mark.parametrize("n", [13000, 40000])
def test_evict_long_sequences(n):
    c = Case([1], [n], 2, 1, 256, 8, seed=5)
    _check_evict(c, _mass(c), 5000, 4, 100)


@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (5, 1), (32, 1)])
def test_mass_with_a_hint_that_is_too_small(heads):
    """More rows than the call was told of: several rounds of the kernel for few rows."""
    c = Case([40, 1, 7], [300, 60, 7], *heads, 16, 50, seed=6)
    lse = _lse(c, 90)
    c.max_q = 1
    _check_mass(c, lse, 90)
    _check_mass(c, lse, 90, mass=torch.randn(3, heads[1], 350, device="cuda").abs())


@pytest.mark.parametrize("window", [-1, 37, 400])
def test_mass_of_single_tokens_over_many_turns(window):
    c = Case([1] * 3, [2500, 17, 1023], 8, 2, 64, 130, seed=7)
    _check_mass(c, _lse(c, window), window)


@pytest.mark.parametrize("window", [-1, 37])
@pytest.mark.parametrize("batch,most", [(40, 700), (600, 90)])  # 600: more than a block counts at once
def test_mass_of_single_tokens_of_many_sequences(batch, most, window):
    rng = np.random.default_rng(batch)
    n_k = [int(n) for n in rng.integers(0, most, batch)]
    n_q = [int(n) for n in rng.integers(0, 3, batch)]
    n_k[7], n_k[-1], n_q[7], n_q[-1] = 4 * most, 3 * most, 1, 2
    c = Case(n_q, n_k, 4, 2, 16, 50, seed=16)
    lse = _lse(c, window)
    _check_mass(c, lse, window)
    _check_mass(c, lse, window, _mass(c))


def test_chunks_of_scores_and_attention():
    """More tokens than a block of rows, windows that begin inside a block's pages."""
    c = Case([70, 33], [900, 40], 8, 2, 16, 60, seed=8)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    for window in (-1, 300):
        got = inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, c.max_q, 60, 16, (window, 0),
                                     block_table=c.table, softmax_scale=c.scale, first_pages=2,
                                     last_pages=1)
        _check_scores(got, *oracle.page_scores(np_(c.q), np_(bounds), np_(c.rel), np_(c.cu_q),
                                               np_(c.cu_k), np_(c.table), 16, 60, window, c.scale, 2, 1))
        check_attention(c, choose(c, 7), window)


def test_wide_tables_and_more_first_and_last_pages_than_there_are():
    c = Case([1], [130], 4, 2, 16, 60, seed=9, extra_columns=3000)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    for first, last in ((2 ** 31 - 1, 0), (0, 2 ** 31 - 1), (3, 2)):
        got = inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 60, 16, block_table=c.table,
                                     softmax_scale=c.scale, first_pages=first, last_pages=last)
        _check_scores(got, *oracle.page_scores(np_(c.q), np_(bounds), np_(c.rel), np_(c.cu_q),
                                               np_(c.cu_k), np_(c.table), 16, 60, -1, c.scale, first,
                                               last))


def test_offsets_that_pass_32_bits():
    """Pages 2^30 + 64 elements apart: the last ones lie beyond 2^32 bytes, and 2^31 elements."""
    c = Case([1, 1], [30, 17], 4, 2, 16, 20, seed=10, spare_pages=0)
    apart = (1 << 30) + 64
    big = [torch.empty(apart * c.pages, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def spread(t, at):
        far = at.as_strided(t.shape, (apart,) + tuple(t.stride()[1:]))
        far.copy_(t)
        return far

    k, v = spread(c.k, big[0]), spread(c.v, big[1])
    near = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    bounds = torch.empty(1 << 31, dtype=torch.bfloat16, device="cuda").as_strided(
        (c.pages, 2, 2, 128), ((1 << 30) // 2, 256, 128, 1))
    inkling_kv_page_bounds(k, c.table, c.cu_k, c.cu_k, bounds=bounds)
    assert torch.equal(bounds, near)
    c.k, c.v = k, v
    _step(c, bounds)
    check_attention(c, choose(c, 2))
    _check_mass(c, _lse(c, -1))
    _check_evict(c, _mass(c), 12, 1, 3)


def test_written_tensors_raise_their_versions_and_tracing_is_refused():
    c = Case([1], [50], 4, 2, 16, 20, seed=11)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    lse, mass = _lse(c, -1), _mass(c)
    old = [t._version for t in (bounds, mass, c.k, c.v)]
    inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k, bounds=bounds)
    inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, 1, 50, 20, block_table=c.table,
                              mass=mass)
    inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, 20)
    assert all(t._version > o for t, o in zip((bounds, mass, c.k, c.v), old))
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda x: inkling_kv_select_pages(x, 2))(torch.zeros(1, 1, 4, device="cuda"))
    with torch.inference_mode():
        x = torch.zeros(c.pages, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
        inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k, bounds=x)


def test_through_the_c_abi_alone(monkeypatch):
    """The same calls without the operator library (argument checks, ctypes)."""
    monkeypatch.setattr(_ops, "USE_TORCH_OPS", False)
    test_the_same_every_time()
    c = Case([3, 1], [200, 150], 8, 2, 16, 64, seed=12, padding=2)
    check_attention(c, choose(c, 5), num_splits=9)
    _check_mass(c, _lse(c, -1))
    _check_evict(c, _mass(c), 100, 1, 64)


def test_python_refusals():
    c = Case([1], [50], 4, 2, 16, 20, seed=13)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    pages = choose(c, 2)
    lse = torch.zeros(4, 1, device="cuda")
    mass = _mass(c)

    def bad(exception, match, f, *a, **kw):
        with pytest.raises(exception, match=match):
            f(*a, **kw)

    B, S, P = inkling_kv_page_bounds, inkling_kv_page_scores, inkling_kv_select_pages
    bad(TypeError, "bfloat16", B, c.k.float(), c.table, c.cu_q, c.cu_k)
    bad(ValueError, "power of two", B, c.k[:, :15], c.table, c.cu_q, c.cu_k)
    bad(ValueError, "unit last stride", B, c.k.transpose(2, 3).contiguous().transpose(2, 3), c.table,
        c.cu_q, c.cu_k)
    bad(ValueError, "bounds must be", B, c.k, c.table, c.cu_q, c.cu_k, bounds=bounds[:, :1])
    bad(ValueError, "block_table", B, c.k, c.table.repeat(2, 1), c.cu_q, c.cu_k)
    bad(TypeError, "int32", B, c.k, c.table, c.cu_q.long(), c.cu_k)
    bad(ValueError, "differ in length", B, c.k, c.table, c.cu_q, torch.cat((c.cu_k, c.cu_k[-1:])))
    kw = dict(block_table=c.table)
    bad(ValueError, "page_size", S, c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 20, 24, **kw)
    bad(ValueError, "rel_extent", S, c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 24, 16, **kw)
    bad(ValueError, "negative", S, c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 20, 16, first_pages=-1, **kw)
    bad(ValueError, "softmax_scale", S, c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 20, 16,
        softmax_scale=0.0, **kw)
    bad(ValueError, "overlap", S, c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 20, 16,
        out=torch.zeros(1, 1, c.width, device="cuda").expand(1, 2, c.width), **kw)
    bad(ValueError, "n_heads", S, c.q[:, :3], bounds, c.rel[:, :3], c.cu_q, c.cu_k, 1, 20, 16, **kw)
    bad(ValueError, "num_selected", P, torch.zeros(1, 1, 4, device="cuda"), 0)
    bad(TypeError, "float32", P, torch.zeros(1, 1, 4, device="cuda").half(), 1)
    D = inkling_fa4_rel_attention_decode_pages
    args = (c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, 50, 20)
    bad(ValueError, "pages must be", D, *args, pages[:, :1], **kw)
    bad(TypeError, "int32", D, *args, pages.long(), **kw)
    bad(ValueError, "block_table", D, *args, pages, block_table=None)
    bad(_lib.Ifa4Error, "num_splits", D, *args, pages, num_splits=-1, **kw)
    bad(ValueError, "workspace", D, *args, pages, workspace=torch.zeros(4, 4, device="cuda").t(), **kw)
    M = inkling_kv_attention_mass
    args = (c.q, c.k, c.rel)
    more = (c.cu_q, c.cu_k, 1, 50, 20)
    bad(ValueError, "lse must be", M, *args, lse.t(), *more, **kw)
    bad(ValueError, "mass must be", M, *args, lse, *more, mass=mass[:, :1], **kw)
    bad(ValueError, "overlap", M, *args, lse, *more, mass=mass[:, :1].expand(1, 2, mass.shape[2]), **kw)
    E = inkling_kv_evict
    bad(ValueError, "budget", E, c.k, c.v, mass, c.table, c.cu_k, 0)
    bad(ValueError, "budget", E, c.k, c.v, mass, c.table, c.cu_k, 10, first=6, recent=5)
    bad(ValueError, "same memory", E, c.k, c.k, mass, c.table, c.cu_k, 10)
    bad(ValueError, "shape", E, c.k, c.v[:-1], mass, c.table, c.cu_k, 10)
    bad(TypeError, "float32", E, c.k, c.v, mass.double(), c.table, c.cu_k, 10)


def test_written_memory_that_overlaps_and_scales_that_are_not_finite_are_refused():
    c = Case([1], [50], 4, 2, 16, 20, seed=14)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    pages, lse, mass = choose(c, 2), _lse(c, -1), _mass(c)
    kw = dict(block_table=c.table, softmax_scale=math.inf)
    with pytest.raises(ValueError, match="softmax_scale"):
        inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, 1, 20, 16, **kw)
    with pytest.raises(ValueError, match="softmax_scale"):
        inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, 1, 50, 20, **kw)
    with pytest.raises(ValueError, match="softmax_scale"):
        inkling_fa4_rel_attention_decode_pages(c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 1, 50, 20, pages,
                                               **kw)
    # a head's maxima in the place of the next one's minima; tokens of one page in the place of the next's
    flat = torch.zeros(c.pages * 768, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.Ifa4Error, match="overlap"):
        inkling_kv_page_bounds(c.k, c.table, c.cu_q, c.cu_k,
                               bounds=flat.as_strided((c.pages, 2, 2, 128), (512, 128, 128, 1)))
    before = c.k.clone()
    k = c.k.as_strided((c.pages - 1, 16, 2, 128), (128, 256, 128, 1))
    with pytest.raises(_lib.Ifa4Error, match="overlap"):
        inkling_kv_evict(k, c.v[:-1], mass, c.table, c.cu_k, 10)
    assert torch.equal(c.k.view(torch.int16), before.view(torch.int16))  # NaN in unused slots


@pytest.mark.parametrize("heads", [4, 40])  # streamed keys, tiles of rows
def test_a_window_as_long_as_it_can_be_is_none(heads):
    c = Case([6, 2, 1], [3, 90, 0], heads, 2, 16, 20, seed=15)  # the first rows lie before every key
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    pages, lse = choose(c, 3), _lse(c, -1)

    def run(window):
        kw = dict(block_table=c.table)
        return (inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, 6, 20, 16, window, **kw),
                inkling_fa4_rel_attention_decode_pages(c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 6, 90, 20,
                                                       pages, window, **kw),
                inkling_kv_attention_mass(c.q, c.k, c.rel, lse, c.cu_q, c.cu_k, 6, 90, 20, window, **kw))

    want = run((-1, -1))
    assert torch.isfinite(want[0]).any() and want[2].any()
    for window in (2**31 - 1, 2**31 - 2, 2**40):
        for x, y in zip(run((window, 0)), want):
            assert torch.equal(x, y)


def test_no_wait_was_given_up():
    assert _lib.read_device_status(torch.cuda.current_stream().cuda_stream, clear=False) == 0
