"""dwarf_amd -- MI355X-native (gfx950) DSQG fixed-offset sparse attention.

Forward, backward and a ring-buffer decode step are HIP kernels in libdsqg_hip.so (C ABI:
include/dsqg.h), exposed as torch custom ops (``dwarf::dsqg_fwd``, ``dwarf::dsqg_bwd``,
``dwarf::dsqg_decode``) and wrapped with the reference's call signatures; so is the block's
interference pool (``dwarf::pool_gate_fwd`` / ``_bwd``), and full attention over a paged key/value
cache (``dwarf::paged_kv_write`` / ``paged_kv_read`` / ``paged_decode`` / ``paged_tree``), and what chooses tokens
(``dwarf::sample_tokens``, ``dwarf::tree_accept``); attention within a window has gradients
(``dwarf::window_fwd`` / ``_bwd``).
"""

from .offsets import ALL_OFFSETS, OFFSETS_V3, OFFSETS_J46, OFFSETS_J47
from .api import (dsqg_attention, dsqg_attention_qkv, dsqg_attention_v2, dsqg_attention_v3,
                  dsqg_attention_backend, dsqg_attention_with_lse, dsqg_decode_step,
                  causal_mean_pool_gate, DSQGRingCache,
                  paged_decode_step, paged_kv_read, paged_kv_write, PagedKVCache,
                  paged_tree_step, draft_tree_accept, sample_tokens, window_attention)
from .modules import DSQGAttentionV3, DSQGAttentionQW, DSQGAttentionN_Fused, DSQGBlock, FFN
from .generation import CondMTransformer, FullAttentionBlock, FullCausalAttention

__all__ = ["ALL_OFFSETS", "OFFSETS_V3", "OFFSETS_J46", "OFFSETS_J47", "dsqg_attention",
           "dsqg_attention_qkv",
           "dsqg_attention_v2", "dsqg_attention_v3", "dsqg_attention_backend",
           "dsqg_attention_with_lse", "dsqg_decode_step", "causal_mean_pool_gate",
           "DSQGRingCache", "paged_decode_step", "paged_kv_read", "paged_kv_write", "PagedKVCache",
           "paged_tree_step", "draft_tree_accept", "sample_tokens", "window_attention",
           "DSQGAttentionV3", "DSQGAttentionQW", "DSQGAttentionN_Fused",
           "DSQGBlock", "FFN", "CondMTransformer", "FullAttentionBlock", "FullCausalAttention"]
