"""The serving steps over a long cache that INTEGRATION.md shows, run as they stand there."""
import os
import re

import numpy as np
import pytest
import torch

import inkling_fa4
from conftest import REPO
from long_context_cases import Case, np_
from test_gpu_page_sparse import check_attention

pytestmark = pytest.mark.gpu


def test_the_long_context_steps():
    text = open(os.path.join(REPO, "INTEGRATION.md")).read()
    block, = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "inkling_kv_evict(" in b]
    sparse, dense = block.split("\n\n")
    c = Case([1, 1], [700, 300], 8, 2, 16, 64, seed=51)
    c.scale = 1 / 128  # the calls name none
    new = [torch.randn(2, 2, 128, device="cuda").to(torch.bfloat16) for _ in range(2)]
    names = {n: getattr(inkling_fa4, n) for n in inkling_fa4.__all__}
    names.update(q=c.q, k=new[0], v=new[1], k_cache=c.k, v_cache=c.v, block_table=c.table, cu_q=c.cu_q,
                 cu_k=c.cu_k, rel=c.rel, R=64, page_size=16, max_k=700, inv_freq=None,
                 bounds=inkling_fa4.inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k),
                 mass=torch.zeros(2, 2, c.width * 16, device="cuda"))
    exec(sparse, names)
    c.q = names["q"]
    check_attention(c, names["pages"], got=names["out"])
    exec(dense, names)
    everything = torch.arange(c.width, dtype=torch.int32, device="cuda").expand(2, 2, c.width)
    check_attention(c, everything, got=names["out"])
    # one query a sequence: its four heads' weights of each KV head sum to one each; 700 weights, each
    # with an exponent and an lse good to 2^-12
    np.testing.assert_allclose(np_(names["mass"]).sum(-1), 4.0, rtol=2.0 ** -11)
