"""Inputs of the long-context tests: sequences of given query and key counts over a paged cache whose
pages lie in random order, with NaN in every slot that no sequence has filled."""
import numpy as np
import torch

EPS32 = 2.0 ** -24  # half a step of fp32, relative
BF16 = 2.0 ** -8    # half a step of bf16, relative
SHAPES = [(4, 4), (8, 2), (12, 4), (5, 1)]


def cu(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32)


class Case:
    """Tensors on `device`; `np_` gives one as float64 (or integers) on the host."""

    def __init__(self, n_q, n_k, heads, kv_heads, page_size, rel_extent, seed=0, padding=0,
                 spare_pages=3, extra_columns=2, device="cuda", merged=False, rel_broadcast=False):
        g = torch.Generator().manual_seed(seed)
        self.n_q, self.n_k = list(n_q), list(n_k)
        self.heads, self.kv_heads, self.page_size, self.rel_extent = heads, kv_heads, page_size, rel_extent
        T, B = sum(n_q) + padding, len(n_q)
        per = [-(-n // page_size) for n in n_k]
        pages = sum(per) + spare_pages
        order = torch.randperm(pages, generator=g)
        width = max(per + [1]) + extra_columns
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(per):
            self.table[b, :c] = order[at:at + c].to(torch.int32)
            at += c

        def bf16(*shape, std=1.0):
            return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)

        self.k, self.v = (bf16(pages, page_size, kv_heads, 128) for _ in range(2))
        filled = torch.zeros(pages, page_size, dtype=torch.bool)
        for b, n in enumerate(n_k):
            for c in range(per[b]):
                filled[self.table[b, c], :min(page_size, n - c * page_size)] = True
        for c in (self.k, self.v):
            c[~filled] = float("nan")
        self.q = bf16(T, heads, 128)
        if merged:  # slices of one projection's output
            both = bf16(T, (heads + 2) * 128)
            self.q = both[:, 128:(heads + 1) * 128].view(T, heads, 128)
        self.rel = bf16(1 if rel_broadcast else T, heads, rel_extent + 3)
        if rel_broadcast:
            self.rel = self.rel.expand(T, heads, rel_extent + 3)
        self.cu_q, self.cu_k = cu(n_q), cu(n_k)
        self.scale = 128 ** -0.5
        self.total, self.pages, self.width = T, pages, width
        for nm in ("q", "k", "v", "rel", "table", "cu_q", "cu_k"):
            t = getattr(self, nm)
            setattr(self, nm, t.to(device) if not rel_broadcast or nm != "rel"
                    else t[:1].to(device).expand(t.shape))
        self.max_q, self.max_k = max(list(n_q) + [1]), max(list(n_k) + [1])


def np_(t):
    t = t.detach().cpu()
    return t.double().numpy() if t.is_floating_point() else t.numpy()
