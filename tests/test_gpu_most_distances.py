"""More distances than the kernels count in 32 bits are refused by every entry point that takes a bias (an
extent of 2^32 + 16 was taken for 16).  The bias is an expanded number; it is refused before it is copied."""
import pytest
import torch

from inkling_fa4 import (_ops, inkling_fa4_rel_attention_decode_pages, inkling_kv_attention_mass,
                         inkling_kv_page_scores)
from long_context_cases import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("extent", [(1 << 29) + 1, (1 << 32) + 16])
def test_refused(extent, path):
    c = Case([1], [30], 2, 1, 16, 8, seed=71)
    rel = c.rel[:, :, :1].expand(1, 2, extent)
    bounds = torch.zeros(c.pages, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(1, 1, 1, dtype=torch.int32, device="cuda")
    lse, kw = torch.zeros(2, 1, device="cuda"), dict(block_table=c.table)
    was = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        for call in (
                lambda: inkling_kv_page_scores(c.q, bounds, rel, c.cu_q, c.cu_k, 1, extent, 16, **kw),
                lambda: inkling_fa4_rel_attention_decode_pages(c.q, c.k, c.v, rel, c.cu_q, c.cu_k, 1, 30,
                                                               extent, pages, **kw),
                lambda: inkling_kv_attention_mass(c.q, c.k, rel, lse, c.cu_q, c.cu_k, 1, 30, extent, **kw)):
            with pytest.raises(ValueError, match="rel_extent"):
                call()
    finally:
        _ops.USE_TORCH_OPS = was
