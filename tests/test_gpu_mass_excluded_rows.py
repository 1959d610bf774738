"""Rows whose lse is -inf add nothing to the gathered weight, whatever their queries, their biases and the
keys that only they see hold (padding of a batch: a caller sets their lse), in every kernel and on every
path through it."""
import numpy as np
import pytest
import torch

from long_context_cases import Case
from test_gpu_kv_evict import _check_mass, _lse

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(8, 2), (12, 4), (5, 1), (16, 4)])
@pytest.mark.parametrize("n_q,n_k", [([1, 3], [200, 90]), ([9, 2], [300, 17]), ([20, 60], [700, 333]),
                                     ([300, 130], [700, 130])])
@pytest.mark.parametrize("extent,window", [(20, -1), (400, -1), (20, 150)])
def test_rows_without_an_lse(extent, window, n_q, n_k, heads):
    c = Case(n_q, n_k, *heads, 16, extent, seed=31, padding=2)
    lse = _lse(c, window)
    rng = np.random.default_rng(1)
    values = (float("nan"), float("inf"), 3e38)
    for t in range(c.total):
        if rng.random() < 0.2 or t == c.total - 3:
            c.q[t] = values[t % 3]
            if t % 2:
                c.rel[t] = values[t % 3]
            lse[:, t] = float("-inf")
    for b in range(2):  # padding at the end: keys that only such rows see
        for i in range(1, min(2, n_q[b]) + 1):
            lse[:, sum(n_q[:b + 1]) - i] = float("-inf")
            at = n_k[b] - i
            c.k[c.table[b, at // 16].long(), at % 16] = float("nan")
    h = int(rng.integers(heads[0]))  # one head of a token only
    c.q[0, h], lse[h, 0] = float("nan"), float("-inf")
    _check_mass(c, lse, window)
