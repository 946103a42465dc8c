"""Importing this package registers the single ``hip`` backend of every op."""

from . import (  # noqa: F401
    attn_decode,
    fused_o_proj_ffn,
    fused_qk_norm_rope,
    gemv,
    kv_cache_quant,
    linear_attn,
    paged_batch_plan,
    qk_norm_mrope,
    quant_attn,
    qwen3_dense_decode,
    reduce,
    rmsnorm,
    softmax,
)
