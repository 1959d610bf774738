"""Workspaces of the shared-prefix decode at every alignment it takes: a buffer that starts 16 bytes
behind a 32-byte boundary (a slice of a pool) gives what an aligned one gives, and nothing in front of
it or behind it is written."""
import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import _ops, inkling_fa4_rel_attention_decode_shared_prefix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("splits", [dict(num_splits=1), dict(num_splits=3, chunk_len=64)],
                         ids=["merged", "split"])
@pytest.mark.parametrize("batch", [3, 70])  # one row tile a KV head, and pairs of them
def test_any_16_byte_alignment(batch, splits, path):
    g = torch.Generator(device="cuda").manual_seed(batch)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)

    prefix, page, own = 300, 16, [1 + 37 * b % 200 for b in range(batch)]
    shared, width = prefix // page, -(-(prefix + 200) // page)
    table = torch.arange(batch * width, dtype=torch.int32, device="cuda").view(batch, width)
    table[:, :shared] = table[0, :shared].clone()
    kc, vc = (randn(batch * width, page, 2, 128) for _ in range(2))
    tail = table[:, shared].long()  # the page in which the prefix ends is each sequence's own copy
    for c in (kc, vc):
        c[tail, :prefix % page] = c[tail[0], :prefix % page].clone()
    lens = torch.tensor([prefix + n for n in own])
    cu_k = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0))).int().cuda()
    cu_q = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    q, rel = randn(batch, 8, 128), randn(batch, 8, 64)
    size = 4 << 20
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        outs = []
        for offset in (0, 16, 32, 48):
            pool = torch.full((size + 128,), 0xff, dtype=torch.uint8, device="cuda")
            assert pool.data_ptr() % 32 == 0
            ws = pool[offset:offset + size]
            outs.append(inkling_fa4_rel_attention_decode_shared_prefix(
                q, kc, vc, rel, cu_q, cu_k, 1, int(lens.max()), 64, prefix, block_table=table,
                prefix_splits=2, workspace=ws, **splits))
            used = pool != 0xff
            assert bool(used.any()) and not bool(used[:offset].any()) and not bool(used[offset + size:].any())
        assert all(torch.equal(outs[0], o) for o in outs[1:])
    finally:
        _ops.USE_TORCH_OPS = before
    assert device_status_ok(), "a kernel abandoned a bounded wait"
