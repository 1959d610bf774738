"""Logits that are no numbers among a sequence's own keys: behind a shared prefix they make the rows
that see them NaN, as the formula does, whatever the plan is (own keys merged with the prefix in one
kernel, or split), and no other row."""
import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import inkling_fa4_rel_attention_decode_shared_prefix

pytestmark = pytest.mark.gpu

PREFIX, PAGE = 128, 16


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


def _batch(own):
    g = torch.Generator().manual_seed(sum(own))

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16).cuda()

    width = PREFIX // PAGE + -(-max(own) // PAGE)
    table = torch.arange(len(own) * width, dtype=torch.int32).view(len(own), width).contiguous()
    table[:, :PREFIX // PAGE] = table[0, :PREFIX // PAGE].clone()
    kc, vc = (randn(len(own) * width, PAGE, 2, 128) for _ in range(2))
    return randn(len(own), 8, 128), kc, vc, randn(len(own), 8, 64), table


def _slot(table, b, key):
    return int(table[b, (PREFIX + key) // PAGE]), (PREFIX + key) % PAGE


def _run(q, kc, vc, rel, table, own, **kw):
    cu_q = torch.arange(len(own) + 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([PREFIX + n for n in own])
    cu_k = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0))).int().cuda()
    return inkling_fa4_rel_attention_decode_shared_prefix(
        q, kc, vc, rel, cu_q, cu_k, 1, int(lens.max()), 64, PREFIX, block_table=table.cuda(),
        return_lse=True, **kw)


# the sequence that gets them, the keys, and the plan of the own keys
@pytest.mark.parametrize("splits", [{}, dict(num_splits=1), dict(num_splits=3, chunk_len=64)],
                         ids=["auto", "one", "three"])
@pytest.mark.parametrize("own,b,keys", [
    ([1, 1, 1], 1, [0]),                        # the only own key
    ([5, 40, 300], 2, [7]),                     # one of many
    ([5, 40, 300], 2, [299]),                   # the newest
    ([5, 40, 300], 1, list(range(40))),         # all of them
    ([200, 40, 300], 0, list(range(64, 128))),  # one whole tile, all four warps' keys
])
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
def test_own_keys(splits, own, b, keys, value):
    q, kc, vc, rel, table = _batch(own)
    for key in keys:
        page, slot = _slot(table, b, key)
        kc[page, slot, 1, 5] = value    # KV head 1
        if value == float("inf"):       # its products are +inf, not -inf
            q[b, 4:, 5] = q[b, 4:, 5].abs() + 1
    out, lse = _run(q, kc, vc, rel, table, own, **splits)
    other = [i for i in range(len(own)) if i != b]
    assert bool(torch.isnan(out[b, 4:].float()).all()) and bool(torch.isnan(lse[4:, b]).all())
    assert bool(torch.isfinite(out[b, :4].float()).all())
    assert bool(torch.isfinite(out[other].float()).all()) and bool(torch.isfinite(lse[:, other]).all())


@pytest.mark.parametrize("splits", [{}, dict(num_splits=3, chunk_len=64)], ids=["auto", "three"])
def test_own_bias(splits):
    """A NaN in the bias of the newest key reaches its row only; +inf gives NaN as well, -inf hides
    the key."""
    own = [5, 40, 300]
    q, kc, vc, rel, table = _batch(own)
    rel[2, 3, 0] = float("nan")
    rel[1, 6, 0] = float("inf")
    rel[0, 2, 0] = -float("inf")
    out, lse = _run(q, kc, vc, rel, table, own, **splits)
    bad = torch.zeros(3, 8, dtype=torch.bool)
    bad[2, 3] = bad[1, 6] = True
    assert torch.equal(torch.isnan(out.float()).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(out.float()).any(-1).cpu(), bad)
    assert torch.equal(torch.isnan(lse.t()).cpu(), bad)


@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("batch", [3, 70])
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("key", [0, 513, 517, 899])
def test_prefix_keys(key, value, batch, splits):
    """The same among the shared keys: in tiles of every kind (the first, interior ones, whose
    exponentials are taken without a row maximum and in part by a polynomial, the last)."""
    prefix, width = 1000, 64
    g = torch.Generator().manual_seed(key)

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16).cuda()

    kc, vc, q, rel = randn(70, 16, 2, 128), randn(70, 16, 2, 128), randn(batch, 8, 128), \
        randn(batch, 8, 64)
    kc[key // 16, key % 16, 0, 7] = value
    q[:, :4, 7] = q[:, :4, 7].abs() + 1
    table = torch.arange(width, dtype=torch.int32, device="cuda").expand(batch, width).contiguous()
    cu_q = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    out, lse = inkling_fa4_rel_attention_decode_shared_prefix(
        q, kc, vc, rel, cu_q, cu_q * (prefix + 5), 1, prefix + 5, 64, prefix, block_table=table,
        prefix_splits=splits, return_lse=True)
    assert bool(torch.isnan(out[:, :4].float()).all()) and bool(torch.isnan(lse[:4]).all())
    assert bool(torch.isfinite(out[:, 4:].float()).all()) and bool(torch.isfinite(lse[4:]).all())
