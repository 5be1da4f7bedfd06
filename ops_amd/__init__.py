"""ops_amd — MI355X (gfx950) top-k sparse flash attention.

Public API (BSHD, see ``ops_amd.sfa``)::

    out, lse = ops_amd.sparse_flash_attention(q, k, v, topk_idxs, sm_scale=None,
                                              kv_lens=None, attn_sink=None)

Paged KV cache (serving): ``ops_amd.sfa_forward_paged(q, k_cache, v_cache,
block_table, topk_idxs, ...)``.

Top-k index producer (scores + selection that create ``topk_idxs``):
``ops_amd.indexer_topk(q_idx, k_idx, weights, topk, kv_lens=None)``.

Around the attention: rotary positions and per-head norms (``ops_amd.rotary_embedding``,
``ops_amd.qk_norm_rope``, and ``ops_amd.qk_norm_rope_append`` into a cache's pages),
dense attention of chunks over the cache (``ops_amd.chunk_attention_paged``) and of
whole sequences (``ops_amd.window_attention``), drafted trees over the cache
(``ops_amd.tree_attention_paged``), and its pages (``ops_amd.cache_extend``,
``cache_fork``, ``cache_free``, ``cache_compact``, ``cache_copy_pages``,
``cache_keep_path``, ``cache_read``).

The HIP kernels live in ``libsfa.so`` (``python -m ops_amd.build``), reached
through the C ABI declared in ``include/sfa.h``.
"""
from .cache import (cache_compact, cache_copy_pages, cache_extend, cache_fork, cache_free,
                    cache_keep_path, cache_read)
from .dense import chunk_attention_paged, window_attention
from .indexer import indexer_topk
from .rope import qk_norm_rope, qk_norm_rope_append, rope_frequencies, rotary_embedding
from .sfa import (SparseFlashAttention, SparseFlashAttentionSBHD, SparseFlashAttentionTriton, sfa_backward,
                  sfa_forward, sfa_forward_paged, sparse_flash_attention)
from .tree import tree_attention_paged

__all__ = ["SparseFlashAttention", "sparse_flash_attention", "sfa_forward", "sfa_backward", "sfa_forward_paged",
           "SparseFlashAttentionSBHD", "SparseFlashAttentionTriton", "indexer_topk",
           "rope_frequencies", "rotary_embedding", "qk_norm_rope", "qk_norm_rope_append", "tree_attention_paged",
           "chunk_attention_paged", "window_attention",
           "cache_copy_pages", "cache_fork", "cache_free", "cache_extend", "cache_compact", "cache_keep_path", "cache_read"]
