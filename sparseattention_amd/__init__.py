"""MI355X-native block-sparse attention forward.

Same Python surface as tomatillos/sparseattention for its one hot path:

* :func:`sparse_attention` (reference: ``sparseattention/sparse_attn_kernel.py:149``)
* :func:`sparse_attention_decode`: the same function for Sq <= 32 with a split-KV launch (the reference names
  decode kernels as future work, ``README.md:65``)
* :func:`sparse_attention_decode_paged`: the same over a K/V cache in pages of 8-bit numbers (:class:`PagedCache`), with the
  operators that store, read back, copy, fork, compact and free its pages
* :func:`rotate_heads`, :func:`rotate_heads_trainable`: norms of queries and keys and their rotation by position in front of attention
* :func:`paged_cache_append_rotated`, :func:`sparse_attention_decode_tree`, :func:`verify_drafts`, :func:`paged_cache_keep`: a step
  with trees of drafted tokens over the paged cache (drafts.py)
* :func:`compute_mask_kernel`, :func:`compute_mask_slow`, :class:`MaskMetadata`
  (reference: ``sparseattention/mask_utils.py:85``, ``:14``, ``:6``)
* :func:`compute_mask_terms`: the same metadata for masks given by a formula (:class:`MaskTerm`), without the
  Sq x Sk tensor (the reference names algebraic masks as future work, ``README.md:63``)

The device work is done by hand-written gfx950 HIP kernels in ``libsparseattn_hip.so``
behind the C ABI of ``include/sparseattn.h``.
"""
from .drafts import verify_drafts
from .mask_utils import (MaskMetadata, MaskTerm, block_term, causal_term, compute_mask_kernel, compute_mask_slow,
                         compute_mask_terms, materialize_mask_terms, select_block_sizes, select_tiling, Tiling,
                         with_list_stats)
from .paged_cache import (PagedCache, empty_paged_cache, paged_cache_append, paged_cache_append_rotated, paged_cache_compact, paged_cache_copy,
                          paged_cache_fork, paged_cache_free_pages, paged_cache_gather, paged_cache_keep, sparse_attention_decode_paged,
                          sparse_attention_decode_tree)
from .rotary import Rotary, rotary_frequencies, rotate_heads, rotate_heads_backward, rotate_heads_trainable
from .sparse_attn_kernel import (BackwardMetadata, compute_backward_metadata, compute_backward_metadata_terms,
                                 merge_attention_parts, sparse_attention,
                                 sparse_attention_backward, sparse_attention_decode, sparse_attention_kv_split,
                                 sparse_attention_tiled, sparse_attention_trainable)

__all__ = ["MaskMetadata", "compute_mask_kernel", "compute_mask_slow", "select_block_sizes", "sparse_attention",
           "sparse_attention_decode", "sparse_attention_backward", "sparse_attention_trainable", "BackwardMetadata",
           "compute_backward_metadata", "merge_attention_parts", "sparse_attention_kv_split", "MaskTerm", "causal_term",
           "block_term", "compute_mask_terms", "materialize_mask_terms", "compute_backward_metadata_terms", "select_tiling",
           "Tiling", "sparse_attention_tiled", "with_list_stats", "PagedCache", "empty_paged_cache", "paged_cache_append",
           "paged_cache_gather", "paged_cache_copy", "paged_cache_fork", "paged_cache_compact", "paged_cache_free_pages",
           "sparse_attention_decode_paged", "Rotary", "rotary_frequencies", "rotate_heads", "rotate_heads_backward",
           "rotate_heads_trainable", "paged_cache_append_rotated",
           "sparse_attention_decode_tree", "paged_cache_keep", "verify_drafts"]
