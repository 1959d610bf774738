"""Refusals of the C ABI of the long-context operators that the layouts' own tests do not have."""
import ctypes

import pytest

from inkling_fa4 import _lib
from test_long_context_cpu import (BOUNDS, CACHE, INVALID, QUERY, SEQS, UNSUPPORTED, _decode_pages, _refused,
                                   _set)


@pytest.mark.parametrize("kw", [
    dict(out_stride_h=64), dict(out_stride_t=256), dict(out_stride_t=128, out_stride_h=128),
    dict(lse=256, lse_stride_h=0, lse_stride_t=1), dict(lse=256, lse_stride_h=3, lse_stride_t=0),
    dict(lse=256, lse_stride_h=2, lse_stride_t=1), dict(lse=256, lse_stride_h=-3, lse_stride_t=1)])
def test_outputs_whose_rows_overlap(kw):
    """Rows of 128 and of one number, 3 tokens and 4 heads: blocks would write one another's rows."""
    need = ctypes.c_size_t(0)
    _refused("ifa4_decode_pages_workspace_size", _decode_pages(**kw), INVALID, b"overlap", ctypes.byref(need))
    _refused("ifa4_decode_pages_launch", _decode_pages(**kw), INVALID, b"overlap", None,
             ctypes.c_size_t(0), None)


@pytest.mark.parametrize("kw", [
    dict(out_stride_t=128, out_stride_h=384), dict(out_stride_t=1024, out_stride_h=256),
    dict(lse=256, lse_stride_h=3, lse_stride_t=1), dict(lse=256, lse_stride_h=1, lse_stride_t=4),
    dict(lse=256, lse_stride_h=1, lse_stride_t=14)])
def test_outputs_whose_rows_lie_apart(kw):
    need = ctypes.c_size_t(0)
    assert _lib.lib().ifa4_decode_pages_workspace_size(ctypes.byref(_decode_pages(**kw)),
                                                       ctypes.byref(need)) == 0


@pytest.mark.parametrize("extent", [(1 << 29) + 1, (1 << 31) - 1])
def test_more_distances_than_positions_in_32_bits(extent):
    """Sums of a distance and a position passed 2^31 in the kernels."""
    need = ctypes.c_size_t(0)
    _refused("ifa4_decode_pages_workspace_size", _decode_pages(rel_extent=extent), UNSUPPORTED, b"rel_extent",
             ctypes.byref(need))
    base = {**SEQS, **QUERY, "head_dim": 128, "kv_heads": 2}
    scores = _set(_lib.PageScoresParams(), **{**base, **BOUNDS, "scores": 256, "rel_extent": extent})
    _refused("ifa4_page_scores_launch", scores, UNSUPPORTED, b"rel_extent", None)
    mass = _set(_lib.AttentionMassParams(), **{**base, **CACHE, "mass": 256, "lse": 256, "rel_extent": extent})
    _refused("ifa4_attention_mass_launch", mass, UNSUPPORTED, b"rel_extent", None)
