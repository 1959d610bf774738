"""Every long-context kernel that writes to places it computes has index checks of the debug build, and so
does the choice that three of them share."""
import os
import re

import pytest

from inkling_fa4.build import CSRC

KERNELS = {"ifa4_page_sparse_sm100.cu": ["page_bounds_kernel", "page_scores_kernel", "select_pages_kernel",
                                         "decode_pages_kernel"],
           "ifa4_kv_evict_sm100.cu": ["attention_mass_kernel", "attention_mass_stream_kernel",
                                      "kv_evict_select_kernel", "kv_evict_move_kernel"]}


def _body(text, start):
    """From the first brace at or behind `start` to its partner."""
    at = text.index("{", start)
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i]
    raise AssertionError("no end")


@pytest.mark.parametrize("file,kernel", [(f, k) for f, ks in KERNELS.items() for k in ks])
def test_kernel_has_checks(file, kernel):
    text = open(os.path.join(CSRC, file)).read()
    start = re.search(rf"__global__ [^;{{]*?\b{kernel}\(", text).end()
    assert "IFA4_DBG_CHECK(" in _body(text, start)


@pytest.mark.parametrize("name,least", [("select_largest_long", 1), ("select_largest", 3)])
def test_choice_has_checks(name, least):
    text = open(os.path.join(CSRC, "ifa4_paged.cuh")).read()
    start = re.search(rf"__forceinline__ int {name}\(", text).end()
    assert _body(text, start).count("IFA4_DBG_CHECK(") >= least
