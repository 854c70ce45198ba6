"""B200-native CASTLE attention (causal attention with lookahead keys).

`Castle` is a drop-in for `lookahead_keys_attention.Castle`; `castle_attention`
replaces the reference's `castle_attention_triton` operator.
"""
from .castle import Cache, Castle, ModuleCache, cache_from_buffers
from .ops import (castle_attention, castle_attention_packed, castle_decode_step, castle_embedding, castle_layer_norm,
                  castle_copy_pages, castle_linear_4bit, castle_linear_cross_entropy, castle_pack_4bit, castle_paged_decode_step,
                  castle_quantize_4bit, castle_write_pages, check_status,
                  release_workspaces)
from .serve import Linear4bit, PagedBatch, PagedCache

__all__ = ["Castle", "Cache", "ModuleCache", "cache_from_buffers", "release_workspaces", "castle_attention", "castle_attention_packed", "castle_decode_step", "castle_embedding", "castle_layer_norm",
           "castle_linear_cross_entropy", "castle_paged_decode_step", "castle_write_pages", "castle_copy_pages", "castle_linear_4bit", "castle_pack_4bit",
           "castle_quantize_4bit", "Linear4bit", "PagedCache", "PagedBatch", "check_status"]
