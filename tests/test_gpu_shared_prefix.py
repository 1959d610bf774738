"""Decode behind a shared prefix on the GPU, against the 64-bit oracle and the plain decode.

Tolerance.  With A = sum of softmax weights times |v|: every weight is rounded to bf16 (2^-8 of
itself) before the product with V, and its exponential is good to 7.5e-5, with scores off by far
less than 1e-4 (fp32 sums of 128 products): (2^-8 + 2^-11) A; the output is rounded to bf16 once
(2^-8 of itself); the merge works in fp32.  The log-sum-exp sums unrounded weights: 1e-3."""
import numpy as np
import pytest
import torch

import oracle
from gpu_util import device_status_ok
from inkling_fa4 import (_ops, inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_decode_triton)
from inkling_fa4.workloads import cu_from_lens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


class Batch:
    """Sequences of ``own`` keys behind ``prefix`` shared ones (``own`` None: an unrelated sequence
    of ``alone`` keys), in pages of random order; the page in which the prefix ends is each
    sequence's own copy; every slot without a key is NaN."""

    def __init__(self, prefix, own, heads, kv, R, page, seed=0, scale=128 ** -0.5, alone=0):
        g = torch.Generator().manual_seed(seed)

        def randn(*shape, std=1.0):
            return (std * torch.randn(*shape, generator=g)).to(torch.bfloat16)

        self.prefix, self.page, self.R, self.scale = prefix, page, R, scale
        self.lens = [alone if s is None else prefix + s for s in own]
        B = len(own)
        shared_pages = prefix // page
        n_per = [-(-n // page) - (shared_pages if s is not None else 0)
                 for n, s in zip(self.lens, own)]
        pages = shared_pages + sum(n_per) + 2
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        width = max([-(-n // page) for n in self.lens] + [shared_pages, 1]) + 2
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        shared_k, shared_v = randn(prefix, kv, 128), randn(prefix, kv, 128)
        self.kc = torch.full((pages, page, kv, 128), float("nan"), dtype=torch.bfloat16)
        self.vc = self.kc.clone()
        at = shared_pages
        for b, (n, s) in enumerate(zip(self.lens, own)):
            first = shared_pages if s is not None else 0
            self.table[b, :first] = perm[:first]
            self.table[b, first:first + n_per[b]] = perm[at:at + n_per[b]]
            at += n_per[b]
            kb, vb = randn(n, kv, 128), randn(n, kv, 128)
            if s is not None:
                kb[:prefix], vb[:prefix] = shared_k, shared_v
            j = torch.arange(n)
            pg = self.table[b, j // page].long()
            self.kc[pg, j % page], self.vc[pg, j % page] = kb, vb
        if shared_pages:  # no sequence may have written them
            j = torch.arange(shared_pages * page)
            pg = perm[j // page].long()
            self.kc[pg, j % page], self.vc[pg, j % page] = (shared_k[:len(j)], shared_v[:len(j)])
        self.q, self.rel = randn(B, heads, 128), randn(B, heads, R, std=0.5)
        self.cu_q, self.cu_k = cu_from_lens([1] * B), cu_from_lens(self.lens)

    def cuda(self):
        for nm in ("table", "kc", "vc", "q", "rel", "cu_q", "cu_k"):
            setattr(self, nm, getattr(self, nm).cuda())
        return self

    def run(self, window=-1, **kw):
        args = dict(window_size=(window, 0), softmax_scale=self.scale, block_table=self.table)
        args.update(kw)
        return inkling_fa4_rel_attention_decode_shared_prefix(
            self.q, self.kc, self.vc, self.rel, self.cu_q, self.cu_k, 1, max(self.lens), self.R,
            kw.pop("prefix", self.prefix), **{k: v for k, v in args.items() if k != "prefix"})

    def plain(self, window=-1, **kw):
        return inkling_fa4_rel_attention_decode_triton(
            self.q, self.kc, self.vc, self.rel, self.cu_q, self.cu_k, 1, max(self.lens), self.R,
            window_size=(window, 0), softmax_scale=self.scale, causal_align="bottom_right",
            block_table=self.table, **kw)

    def check(self, window=-1, **kw):
        out, lse = self.run(window, return_lse=True, **kw)

        def np_(t):
            return t.double().cpu().numpy()

        want, want_lse, size = oracle.decode_paged(
            np_(self.q), np_(self.kc), np_(self.vc), np_(self.rel), self.lens,
            self.table.cpu().numpy(), self.scale, self.R, window)
        tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * size
        err = np.abs(np_(out) - want) - tol
        assert err.max() <= 0, f"output: {err.max()}"
        np.testing.assert_allclose(np_(lse), want_lse, atol=1e-3, rtol=0)
        return out, lse


CASES = [  # prefix, own, heads, kv, rel_extent, page, window
    (64, [3], 4, 4, 16, 16, -1),
    (128, [1, 2], 8, 2, 128, 16, -1),
    (300, [0, 1, 5, 130, 64, 0], 8, 2, 100, 16, -1),           # the prefix ends inside a page
    (2048, list(range(1, 34)), 32, 8, 128, 16, -1),            # two tiles: pairs of row tiles
    (1000, [7] * 5, 12, 4, 1000, 32, -1),                      # group of three, a long bias
    (257, [40, 3, 1], 5, 1, 64, 256, -1),                      # group of five, one KV head
    (640, [1] * 70, 4, 4, 128, 64, -1),                        # no grouping: 70 rows
    (512, [9, 100] * 100, 4, 2, 64, 16, -1),                   # 200 sequences, an odd last tile
    (1, [0, 1, 2], 4, 2, 16, 16, -1),
    (16, [0, 0], 4, 2, 16, 16, -1),
    (900, [1, 50, 400], 8, 2, 128, 16, 300),                   # window: parts, all, none of it
    (900, [1, 50, 400], 8, 2, 128, 16, 0),
    (1500, [600, 700], 8, 2, 64, 32, 500),                     # window: no row sees the prefix
    (200, [2, 2, 2], 48, 1, 64, 16, -1),                       # group of 48: two sequences a tile
    (200, [2, 30, 2], 128, 1, 64, 16, -1),                     # group of 128
    (260, [2000, 1, 700], 8, 2, 128, 16, -1),                  # long own keys: split, then merged
    (4000, [0, 1100], 4, 1, 64, 64, -1),                       # more than 32 partials a row
    (3000, [5, 40] * 8, 8, 1, 64, 16, -1),                     # the same, merged in the decode
]


@pytest.mark.parametrize("prefix,own,heads,kv,R,page,window", CASES)
def test_against_oracle(prefix, own, heads, kv, R, page, window):
    b = Batch(prefix, own, heads, kv, R, page, seed=len(own)).cuda()
    b.check(window)


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("splits", [1, 3, 40])
def test_any_plan_and_path(path, splits):
    """Forced prefix splits (more than there are key tiles: most are empty), own-key splits, a
    workspace that is used again, an output and a log-sum-exp buffer."""
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        b = Batch(700, [5, 300, 1, 64], 8, 2, 128, 16, seed=3).cuda()
        ws = torch.full((8 << 20,), 0xff, dtype=torch.uint8, device="cuda")
        for kw in (dict(prefix_splits=splits), dict(prefix_splits=splits, num_splits=3,
                                                    chunk_len=64, workspace=ws)):
            b.check(**kw)
        out = torch.zeros(4, 16, 128, dtype=torch.bfloat16, device="cuda")[:, 4:12]
        lse = torch.zeros(4, 8, device="cuda").t()
        got = b.run(out=out, lse=lse, prefix_splits=splits)
        want = b.run(return_lse=True, prefix_splits=splits)
        assert got[0].data_ptr() == out.data_ptr()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    finally:
        _ops.USE_TORCH_OPS = before


def test_sequences_that_share_nothing():
    """Sequences with fewer keys than the prefix (some empty, the first among them) are attended
    whole through their own pages, whatever the prefix is; an empty one gives 0 and -inf."""
    b = Batch(400, [None, 3, None, 0, 77], 8, 2, 128, 16, seed=5, alone=399).cuda()
    b.check()
    b = Batch(400, [None, 3, 9, None], 8, 2, 128, 16, seed=6, alone=0).cuda()
    out, lse = b.check()
    assert bool((out[0] == 0).all()) and bool((lse[:, 0] == -float("inf")).all())
    b = Batch(400, [None, None], 8, 2, 128, 16, seed=7, alone=100).cuda()
    b.check()  # nobody shares it


def test_prefix_of_zero_is_the_plain_decode():
    b = Batch(200, [5, 300, 1], 8, 2, 128, 16, seed=3).cuda()
    assert torch.equal(b.run(prefix=0), b.plain())


@pytest.mark.parametrize("own", [[700, 650, 610], [610] * 20 + [700] * 60])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_behind_every_window(own, page):
    """Pages that have left a sequence's window may be gone from its table row, and from the cache:
    those no window reaches hold NaN by now.  The windows of the sequences behind the first ones
    reach further back than theirs, or less far (20 + 60 sequences, three row tiles)."""
    prefix, window = 1000, 1000
    b = Batch(prefix, own, 8, 2, 128, page, seed=12)
    live = torch.zeros(b.kc.shape[0], dtype=torch.bool)
    for i, n in enumerate(b.lens):
        first = (n - 1 - window) // page  # the page of the first visible key
        live[b.table[i, first:-(-n // page)].long()] = True
        b.table[i, :first] = -1
    assert not live.all()
    b.kc[~live] = float("nan")
    b.vc[~live] = float("nan")
    b.cuda().check(window)


def test_large_scores_and_masked_values():
    """Scores of several hundred: the running maximum moves between tiles.  The lowest bf16 value
    and -inf as bias hide keys; a row whose bias hides every key it sees gives 0."""
    b = Batch(1000, [20, 1, 5], 8, 2, 1200, 16, seed=8, scale=4.0).cuda()
    b.check()
    b = Batch(300, [20, 1, 5], 8, 2, 512, 16, seed=9)
    b.rel[0, 3, 10:200] = torch.finfo(torch.bfloat16).min
    b.rel[1, 2, 5:290] = -float("inf")
    b.rel[2, 0, 5:] = -float("inf")      # the prefix is hidden whole, the own keys are not
    b.cuda().check()
    b.rel[1, 7] = -float("inf")
    out, lse = b.run(return_lse=True)
    assert bool((out[1, 7] == 0).all()) and float(lse[7, 1]) == -float("inf")
    assert bool(torch.isfinite(out.float()).all())


def test_bias_layouts():
    """A per-head table with token stride 0, an odd offset (scalar reads), a wider tensor."""
    b = Batch(500, [20, 1, 90], 8, 2, 96, 16, seed=10)
    b.rel = b.rel[:1].expand(3, 8, 96)
    b.cuda()
    b.rel = b.rel[:1].expand(3, 8, 96)
    assert b.rel.stride(0) == 0
    b.check()
    wide = torch.randn(3, 8, 105, device="cuda").to(torch.bfloat16)
    for off in (0, 1, 8):
        b.rel = wide[:, :, off:off + 96]
        b.check()


def test_close_to_the_plain_decode_and_the_same_every_time():
    b = Batch(4096, [1 + 13 * i % 500 for i in range(48)], 32, 8, 128, 16, seed=11).cuda()
    got, lse = b.run(return_lse=True)
    want, want_lse = b.plain(return_lse=True)
    torch.testing.assert_close(got.float(), want.float(), atol=4e-3, rtol=2e-2)
    torch.testing.assert_close(lse, want_lse, atol=1e-3, rtol=0)
    again = b.run(return_lse=True)
    assert torch.equal(got, again[0]) and torch.equal(lse, again[1])


def test_refusals():
    b = Batch(64, [3, 1], 8, 2, 16, 16, seed=1).cuda()
    with pytest.raises(ValueError, match="block_table"):
        b.run(block_table=None)
    with pytest.raises(ValueError, match="shared_prefix_len"):
        b.run(prefix=-1)
    with pytest.raises(ValueError, match="beyond the table"):
        b.run(prefix=10000)
    for ws in (torch.zeros(8 << 20, dtype=torch.uint8),  # on the CPU
               torch.zeros(2 << 20, 8, dtype=torch.uint8, device="cuda")[:, ::2]):
        with pytest.raises(ValueError, match="workspace"):
            b.run(workspace=ws)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        b.run(workspace=torch.zeros((8 << 20) + 8, dtype=torch.uint8, device="cuda")[8:])
    with pytest.raises(ValueError, match="one query"):
        inkling_fa4_rel_attention_decode_shared_prefix(
            b.q.repeat(2, 1, 1), b.kc, b.vc, b.rel.repeat(2, 1, 1), b.cu_q, b.cu_k, 1, 67, 16, 64,
            block_table=b.table)
    with pytest.raises(RuntimeError, match="128 query heads"):
        inkling_fa4_rel_attention_decode_shared_prefix(
            torch.zeros(2, 129, 128, dtype=torch.bfloat16, device="cuda"), b.kc[:, :, :1],
            b.vc[:, :, :1], torch.zeros(2, 129, 16, dtype=torch.bfloat16, device="cuda"), b.cu_q,
            b.cu_k, 1, 67, 16, 64, block_table=b.table)
