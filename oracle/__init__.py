"""CPU oracle (test infrastructure only): see ``oracle/rel_attn_oracle.py`` (attention),
``oracle/rel_logits_oracle.py`` (rel_logits producer) and ``oracle/operators_oracle.py`` (the other
operators next to the attention, in 64 bits)."""
from .rel_attn_oracle import (  # noqa: F401
    rel_attn,
    rel_attn_rows,
    round_to_bf16,
    bf16_bits_to_f32,
    f32_to_bf16_bits,
    alignment_offsets,
    rel_attn_torch,
    rel_attn_rows_torch,
    rel_attn_grads_torch,
)
from .rel_logits_oracle import token_positions, log_tau, rel_logits_proj  # noqa: F401
from .operators_oracle import (  # noqa: F401
    norm_rope,
    norm_rope_pair_size,
    norm_rope_grads,
    kv_append,
    decode_paged,
    bucket_of,
    bucket_bias,
    bucket_bias_grad,
)
