"""The check that rows written in place have no element in common with rows read by the same launch,
against the sets of their elements; and that the layouts a layer has pass it."""
import random

import pytest
import torch

from inkling_fa4.qk_norm_rope import _apart


def _elements(t):
    return set((torch.arange(t.untyped_storage().nbytes() // 2)
                .as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()))


def test_never_true_of_rows_that_overlap():
    rng = random.Random(1)
    pool = torch.zeros(6000, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(1500):
        rows = []
        st = rng.choice([256, 384, 512, 1024])
        for _ in range(2):
            shape = (rng.randint(1, 4), rng.randint(1, 3), 128)
            strides = (rng.choice([st, st, 256, 520]), rng.choice([0, 8, 128, 136, 256, 384]), 1)
            span = sum((n - 1) * s for n, s in zip(shape, strides))
            rows.append(pool.as_strided(shape, strides, 8 * rng.randint(0, (5999 - span) // 8)))
        apart = _apart(*rows)
        assert apart == _apart(*rows[::-1])
        seen[apart] += 1
        if apart:
            assert not _elements(rows[0]) & _elements(rows[1])
    assert min(seen.values()) > 100


@pytest.mark.parametrize("tokens", [1, 5])
def test_layouts_of_a_layer(tokens):
    merged = torch.zeros(tokens, 10 * 128, dtype=torch.bfloat16)
    q, k, v = (merged[:, a * 128:b * 128].view(tokens, b - a, 128)
               for a, b in ((0, 6), (6, 8), (8, 10)))
    turns = torch.zeros(tokens, 4, 3, 128, dtype=torch.bfloat16)      # q, k, v of a head in turn
    stacked = torch.zeros(3, tokens, 4, 128, dtype=torch.bfloat16)    # one behind the other
    for a, b, c in ((q, k, v), turns.unbind(2), stacked.unbind(0)):
        assert _apart(a, b) and _apart(a, c) and _apart(c, a)
        assert not _apart(a, a)
    assert not _apart(q, merged[:, 5 * 128:7 * 128].view(tokens, 2, 128))
    assert _apart(q, q.clone()) and _apart(q, q[:0])
