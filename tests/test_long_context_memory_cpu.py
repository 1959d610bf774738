"""Memory that the eviction and the choice refuse: outputs on top of inputs or of one another, caches that
share elements; against the sets of elements.  The C ABI refuses before any CUDA call; of what it
accepts only the workspace's size is asked for, so the addresses are never used."""
import ctypes
import random

import pytest
import torch

from inkling_fa4 import _lib

INVALID = _lib.IFA4_ERR_INVALID_ARGUMENT


def _evict(k, v, kept=1 << 20, cu_out=1 << 21, mass=1 << 22, mass_out=1 << 23, cu_k=1 << 24,
           table=1 << 25, batch=2, **strides):
    """Parameters of an eviction of caches of the layout of the tensors k and v, `at` their addresses."""
    p = _lib.KvEvictParams()
    s = p.seqs
    s.batch, s.page_size, s.num_pages, s.table_width = batch, k.shape[1], k.shape[0], 4
    s.block_table, s.cu_seqlens_k, s.block_table_stride = table, cu_k, 4
    base = 1 << 30
    p.k_cache, p.v_cache = (base + 2 * t.storage_offset() for t in (k, v))
    p.k_stride_page, p.k_stride_t, p.k_stride_h = k.stride()[:3]
    p.v_stride_page, p.v_stride_t, p.v_stride_h = v.stride()[:3]
    p.kv_heads, p.head_dim, p.budget, p.mass_width = k.shape[2], 128, 4, 64
    p.kept, p.cu_out, p.mass, p.mass_out = kept, cu_out, mass, mass_out
    p.mass_stride_b = p.mass_out_stride_b = 64 * k.shape[2]
    p.mass_stride_h = p.mass_out_stride_h = 64
    if not k.shape[0]:
        p.k_cache = p.v_cache = 1 << 20  # no pages: nothing lies there
    for n, x in strides.items():
        setattr(p, n, x)
    return p


def _says(p):
    """The refusal's text, None where the parameters are accepted."""
    need = ctypes.c_size_t(0)
    rc = _lib.lib().ifa4_kv_evict_workspace_size(ctypes.byref(p), ctypes.byref(need))
    if rc == 0:
        return None
    assert rc == INVALID
    text = _lib.lib().ifa4_last_error_string().decode()
    assert _lib.lib().ifa4_kv_evict_launch(ctypes.byref(p), None, ctypes.c_size_t(0), None) == INVALID
    return text


def _caches(kind, pages=3, size=16, heads=2):
    if kind == "two tensors":
        both = torch.empty(2, pages, size, heads, 128, dtype=torch.bfloat16)
        return both[0], both[1]
    if kind == "pages in turn":
        return torch.empty(pages, 2, size, heads, 128, dtype=torch.bfloat16).unbind(1)
    if kind == "tokens in turn":
        return torch.empty(pages, size, 2, heads, 128, dtype=torch.bfloat16).unbind(2)
    if kind == "heads in turn":
        return torch.empty(pages, size, heads, 2, 128, dtype=torch.bfloat16).unbind(3)
    if kind == "one row":
        return torch.empty(pages, size, heads, 256, dtype=torch.bfloat16).split(128, 3)
    both = torch.empty(pages, 2, heads, size, 128, dtype=torch.bfloat16).unbind(1)  # heads before tokens
    return tuple(t.transpose(1, 2) for t in both)


KINDS = ["two tensors", "pages in turn", "tokens in turn", "heads in turn", "one row", "heads first"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pages,heads", [(3, 2), (1, 1), (1, 4), (5, 1)])
def test_caches_that_lie_beside_one_another(kind, pages, heads):
    k, v = _caches(kind, pages, 16, heads)
    assert _says(_evict(k, v)) is None and _says(_evict(v, k)) is None


def _elements(t):
    return set((torch.arange(t.untyped_storage().nbytes() // 2)
                .as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()))


def test_caches_that_share_elements():
    """Every pair of views with the same strides is refused exactly where they have an element in common."""
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    pool = torch.zeros(60000, dtype=torch.bfloat16)
    for _ in range(600):
        shape = (rng.randint(1, 3), 16, rng.randint(1, 3), 128)
        strides, reach = {}, 128
        for d in rng.sample([0, 1, 2], 3):  # which dimension lies innermost
            strides[d] = reach + 8 * rng.choice([0, 0, 1, 16, 17, 32])
            reach = strides[d] * (shape[d] - 1) + reach
        if 2 * reach > 50000:
            continue
        strides = (strides[0], strides[1], strides[2], 1)
        at = rng.randint(0, min(2 * reach, 59000 - reach) // 8) * 8
        k, v = pool.as_strided(shape, strides, 8 * rng.randint(0, 10)), pool.as_strided(shape, strides, at)
        text = _says(_evict(k, v))
        common = bool(_elements(k) & _elements(v))
        assert (text is not None) == common, (shape, strides, k.storage_offset(), at)
        assert text is None or "v_cache" in text
        seen[common] += 1
    assert min(seen.values()) > 50


def test_caches_of_other_strides():
    pool = torch.zeros(40000, dtype=torch.bfloat16)
    k = pool.as_strided((2, 16, 2, 128), (4096, 256, 128, 1), 0)
    other = (2 * 16 * 256, 256, 128, 1)
    assert "v_cache" in _says(_evict(k, pool.as_strided((2, 16, 2, 128), other, 4096)))
    assert _says(_evict(k, pool.as_strided((2, 16, 2, 128), other, 8192))) is None


def test_caches_of_other_strides_in_turn():
    """Keys [token, head] and values [head, token] of a page, page after page."""
    pool = torch.zeros(3, 2, 16 * 2 * 128, dtype=torch.bfloat16)
    k = pool[:, 0].view(3, 16, 2, 128)
    v = pool[:, 1].view(3, 2, 16, 128).transpose(1, 2)
    assert _says(_evict(k, v)) is None and _says(_evict(v, k)) is None
    shifted = v.as_strided(v.shape, v.stride(), v.storage_offset() - 8)
    assert "v_cache" in _says(_evict(k, shifted)) and "v_cache" in _says(_evict(shifted, k))


def test_never_accepts_other_strides_that_share_an_element():
    rng = random.Random(4)
    pool = torch.zeros(60000, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(800):
        shape = (rng.randint(1, 3), 16, rng.randint(1, 3), 128)
        page, views = 2 * 16 * shape[2] * 128 + 8 * rng.choice([0, 16]), []
        for _ in range(2):
            inner = rng.choice([(shape[2] * 128, 128), (128, 16 * 128), (shape[2] * 128 + 8, 128)])
            views.append(pool.as_strided(shape, (page, *inner, 1), 8 * rng.randint(0, 3000)))
        refused = _says(_evict(*views)) is not None
        seen[refused] += 1
        assert refused or not _elements(views[0]) & _elements(views[1])
    assert min(seen.values()) > 50


@pytest.mark.parametrize("what,with_,kw", [
    ("cu_out", "cu_seqlens_k", dict(cu_out=1 << 24)), ("cu_out", "cu_seqlens_k", dict(cu_out=(1 << 24) + 8)),
    ("cu_out", "cu_seqlens_k", dict(cu_out=(1 << 24) - 8)), ("cu_out", "block_table", dict(cu_out=1 << 25)),
    ("cu_out", "kept", dict(cu_out=(1 << 20) + 60)), ("mass_out", "mass", dict(mass_out=(1 << 22) + 4)),
    ("mass_out", "mass", dict(mass_out=(1 << 22) - 252)), ("kept", "mass", dict(kept=(1 << 22) + 64)),
    ("kept", "k_cache", dict(kept=1 << 30)), ("mass_out", "kept", dict(mass_out=1 << 20)),
    ("cu_out", "mass", dict(cu_out=(1 << 22) + 1020)),
    ("cu_out", "v_cache", dict(cu_out=(1 << 30) + 3 * 16 * 2 * 256 + 64))])
def test_outputs_on_top_of_something(what, with_, kw):
    text = _says(_evict(*_caches("two tensors"), **kw))
    assert text is not None and what in text and with_ in text


def test_caches_without_pages():
    k = torch.empty(1, 16, 2, 128, dtype=torch.bfloat16)[:0]
    assert _says(_evict(k, k)) is None


def test_outputs_next_to_something():
    k, v = _caches("two tensors")
    assert _says(_evict(k, v, cu_out=(1 << 24) + 12)) is None
    assert _says(_evict(k, v, cu_out=(1 << 24) - 12)) is None
    assert _says(_evict(k, v, mass_out=(1 << 22) + 2 * 2 * 64 * 4)) is None
    # columns of one tensor
    wide = dict(mass_stride_b=256, mass_stride_h=128, mass_out_stride_b=256, mass_out_stride_h=128)
    assert _says(_evict(k, v, mass_out=(1 << 22) + 64 * 4, **wide)) is None
    assert "mass_out" in _says(_evict(k, v, mass_out=(1 << 22) + 63 * 4, **wide))


def test_a_choice_on_top_of_its_scores():
    p = _lib.SelectPagesParams()
    p.scores, p.rows, p.kv_heads, p.width, p.num_selected = 1 << 20, 2, 2, 64, 8
    p.scores_stride_t, p.scores_stride_h, p.pages_stride_t, p.pages_stride_h = 128, 64, 16, 8
    for p.pages in (1 << 20, (1 << 20) + 1020, (1 << 20) - 92):
        assert _lib.lib().ifa4_select_pages_launch(ctypes.byref(p), None) == INVALID
        assert b"share memory" in _lib.lib().ifa4_last_error_string()
