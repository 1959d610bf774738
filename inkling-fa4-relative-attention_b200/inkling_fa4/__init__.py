"""inkling_fa4 — B200 (sm_100a) relative-position-bias flash attention.

Drop-in for the reference package's call surface (src/inkling_fa4/__init__.py:1-10):
``inkling_fa4_rel_attention_triton`` (prefill / varlen / chunked / sliding window),
``inkling_fa4_rel_attention_decode_triton`` (split-KV decode), ``ref_rel_attn`` (dense PyTorch
statement for tests) and ``autotune_configs``; beyond the reference, the backward
(``inkling_fa4_rel_attention_backward``), a differentiable ``inkling_fa4_rel_attention``, the
fused ``rel_logits`` producer (``inkling_rel_logits``) and the learned bias by distance buckets
(``inkling_bucket_bias``), the norm and rotation of queries and keys (``inkling_qk_norm_rope``), the
append to the paged cache (``inkling_kv_append``) and decode for a batch that shares a prefix
(``inkling_fa4_rel_attention_decode_shared_prefix``).  The kernels are hand-written CUDA for sm_100a
behind the C ABI of include/inkling_fa4.h; there is no Triton and no CPU fallback.
"""
from .triton_kernel import inkling_fa4_rel_attention_triton
from .reference import ref_rel_attn
from . import autotune_configs
from .triton_kernel_decode import inkling_fa4_rel_attention_decode_triton
from .backward import inkling_fa4_rel_attention, inkling_fa4_rel_attention_backward
from .rel_logits import inkling_rel_logits
from .qk_norm_rope import (inkling_kv_append, inkling_qk_norm_rope, inkling_qk_norm_rope_backward)
from .shared_prefix import inkling_fa4_rel_attention_decode_shared_prefix
from .bucket_bias import (inkling_bucket_bias, inkling_bucket_bias_backward,
                          relative_bucket_starts)

__all__ = [
    "inkling_fa4_rel_attention_triton",
    "inkling_fa4_rel_attention_decode_triton",
    "ref_rel_attn",
    "autotune_configs",
    "inkling_fa4_rel_attention",
    "inkling_fa4_rel_attention_backward",
    "inkling_rel_logits",
    "inkling_qk_norm_rope",
    "inkling_qk_norm_rope_backward",
    "inkling_kv_append",
    "inkling_fa4_rel_attention_decode_shared_prefix",
    "inkling_bucket_bias",
    "inkling_bucket_bias_backward",
    "relative_bucket_starts",
]
