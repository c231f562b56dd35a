"""quant_flash_attn_amd -- INT8 per-token quantized flash attention on AMD MI355X (gfx950).

Same Python entry points as yisunlp/quant_flash_attn, backed by hand-written HIP kernels in
libqfa.so (C ABI in include/qfa.h):

    asymmetric_quant_per_token(x)                      -> (codes, scale, zero_point)
    quant_flash_attn(q, kv_fp16, kv_quant, sm_scale)   -> o      (reference entry point)
    quant_flash_attn_qkv(q, k, v, causal, sm_scale)    -> o      (q/k/v entry point, causal flag)
    quant_flash_attn_quantized_kv(q, k_fp16, v_fp16, k_quant, v_quant, causal, sm_scale) -> o
                                                                 (K and V as two INT8 tensors, as a KV cache holds them)
    norm_rope_pair(q, k, q_weight, k_weight, cos, sin)  -> q, k  (RMSNorm of each head and position rotation; norm_rope: one tensor)
    paged_cache_append(cache, k, v, page_table, starts) , quant_flash_attn_paged(q, cache, page_table, starts) -> o
                                                                 (an INT8 cache in pages, sequences of any lengths)
    paged_select_blocks(q, cache, bounds, page_table, starts, keep) , quant_flash_attn_paged_blocks(..., blocks) -> o
                                                                 (attention on the blocks whose bounds promise the most)
    paged_attention_weights(q, cache, lse, page_table, starts) , paged_cache_evict(cache, page_table, lengths, weights, ...)
                                                                 (eviction by accumulated attention weight)

GPU only: a CPU tensor or a missing libqfa.so raises; there is no fallback implementation.
"""
from .asymmetric_quant import (QuantizedTokens, asymmetric_quant_per_token, code_rowsum, dequantize_per_token,
                               quantize_for_attention, quantize_pair_for_attention)
from .quant_flash_attn import (QuantFlashAttention, QuantFlashAttnQKV, attn_bwd_quantized, attn_fwd_quantized,
                               attn_bwd_shared_kv, attn_fwd_shared_kv,
                               QuantFlashAttnQuantizedKV, quant_flash_attn, quant_flash_attn_qkv,
                               quant_flash_attn_quantized_kv)
from .norm_rope import norm_rope, norm_rope_pair, rope_table
from .paged_blocks import (PageBounds, make_page_bounds, paged_bounds_update, paged_select_blocks,
                           quant_flash_attn_paged_blocks)
from .paged_evict import paged_attention_weights, paged_cache_evict
from .paged_cache import PagedCache, make_paged_cache, paged_cache_append, paged_cache_read, quant_flash_attn_paged

__all__ = [
    "QuantizedTokens", "asymmetric_quant_per_token", "code_rowsum", "dequantize_per_token", "quantize_for_attention",
    "quantize_pair_for_attention",
    "QuantFlashAttention", "QuantFlashAttnQKV", "QuantFlashAttnQuantizedKV", "quant_flash_attn", "quant_flash_attn_qkv",
    "quant_flash_attn_quantized_kv",
    "norm_rope", "norm_rope_pair", "rope_table",
    "PagedCache", "make_paged_cache", "paged_cache_append", "paged_cache_read", "quant_flash_attn_paged",
    "PageBounds", "make_page_bounds", "paged_bounds_update", "paged_select_blocks", "quant_flash_attn_paged_blocks",
    "paged_attention_weights", "paged_cache_evict",
    "attn_fwd_quantized", "attn_bwd_quantized", "attn_fwd_shared_kv", "attn_bwd_shared_kv",
]
__version__ = "0.1.0"
