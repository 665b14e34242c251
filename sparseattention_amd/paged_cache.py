"""K/V cache in pages of 8-bit numbers, and few-rows attention over it.

The reference keeps no cache; the attention is its forward (sparse_attn_kernel.py:149-185) for few query rows, as
:func:`sparseattention_amd.sparse_attention_decode` is, with K and V read from pages.  A serving step is

    paged_cache_append(cache, k, v, page_table, lens)                      # the step's tokens
    o = sparse_attention_decode_paged(q, cache, page_table, lens + 1)      # and their attention

and a prompt's later chunk, which has more than 32 rows, reads its keys back:

    paged_cache_append(cache, k, v, page_table, lens)
    K, V = paged_cache_gather(cache, page_table, lens + n)
    K, V = (x.repeat_interleave(q.shape[1] // cache.num_heads, 1) for x in (K, V))
    o = sparse_attention(q, K, V, mask, BLOCK_Q, BLOCK_K)

(sparse_attention has a K/V head per query head: with grouped heads the third line copies K and V for each of a group.)

All calls enqueue work on the current stream of the cache's device and read no tensor on the host, so they can be captured
into a graph (tile lists that a caller wrote or changed are looked at on the host, once, by the first call that gets them).  The steps of a call are native (csrc/host_ops.cpp), the kernels csrc/paged_cache.hip and csrc/paged_decode.hip."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _native
from .mask_utils import MaskMetadata

PAGE_SIZES = (32, 64, 128, 256)
MOST_PAGES = 1 << 20


@dataclass
class PagedCache:
    """A pool of pages (:func:`empty_paged_cache`).  Blocks of 32 consecutive tokens of one head are e4m3 codes with one scale
    2^e each, e the least integer for which the block's largest finite magnitude is at most 448 * 2^e (-96 <= e <= 119): a
    value is off by at most 2^-4 of itself, or by 2^-10 * 2^e where it is smaller than 2^-6 * 2^e.  Where later tokens made the
    scale grow it was rounded again each time, and is off by less than 2^-4 of itself and 2^-9 * 2^e together.  What is larger than 448 * 2^119
    (2.98e38; bf16 ends at 3.39e38) is held as that.  NaN and infinities are held as NaN.

    ``k``, ``v``: uint8 [pages, H, page_size / 32, 32 * D], in the order the kernels read (:func:`paged_cache_gather` gives
    the values); ``k_scales``, ``v_scales``: float32 [pages, H, page_size / 32].  Head dims that the kernels do not have (they have
    64, 128 and 256) are held with zero columns up to the next."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    head_dim: int

    @property
    def num_pages(self) -> int:
        return self.k.shape[0]

    @property
    def num_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return 32 * self.k.shape[2]


def empty_paged_cache(num_pages: int, H: int, D: int, *, page_size: int = 64, device=None) -> PagedCache:
    """A cache of ``num_pages`` pages (at most 2^20) of ``page_size`` (32, 64, 128 or 256) tokens of ``H`` K/V heads with head dim
    ``D`` (up to 256), all zero: 2 * H * page_size * D bytes a page, and 8 bytes of scales per 32 tokens and head."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES} (got {page_size})")
    if not 1 <= num_pages <= MOST_PAGES or H < 1 or not 1 <= D <= 256:
        raise ValueError(f"expected 1..{MOST_PAGES} pages, at least one head and a head dim of 1..256 (got {num_pages}, {H}, {D})")
    if num_pages * H * (page_size // 32) > 0x7FFFFFFF:
        raise ValueError("more than 2^31 - 1 blocks of 32 tokens in the cache")
    device = torch.device("cuda") if device is None else torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("a paged cache needs a ROCm GPU; there is no CPU path")
    Dk = 64 if D <= 64 else 128 if D <= 128 else 256
    codes = [torch.zeros(num_pages, H, page_size // 32, 32 * Dk, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros(num_pages, H, page_size // 32, dtype=torch.float32, device=device) for _ in range(2)]
    return PagedCache(*codes, *scales, int(D))


def paged_cache_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
                       counts: Optional[torch.Tensor] = None) -> None:
    """Stores new tokens: the first ``counts[b]`` (None: all) of ``k``, ``v`` [B,H,S,D] (bf16 or fp16, any strides) become
    tokens ``lens[b]``, ``lens[b] + 1``, ... of sequence ``b``, whose token ``t`` lies in page ``page_table[b, t // page_size]``.

    ``page_table`` int32 [B, pages], ``lens``, ``counts`` int32 [B], on the cache's device; ``lens`` is what the sequences hold before and
    is not changed.  Tokens past the table, and those whose entry is no page, are not stored.  The 32 tokens of a block
    share a scale: one that holds some keeps its scale or takes a larger one, with which what it holds is rounded again;
    what a block held before its first token of the sequence does not count.  Sequences of one call, or two entries of one, must not
    store into the same page (fork it first: :func:`paged_cache_fork`)."""
    _native.host().paged_append(cache, k, v, page_table, lens, counts)


def paged_cache_gather(cache: PagedCache, page_table: torch.Tensor, lens: torch.Tensor, length: Optional[int] = None,
                       dtype: torch.dtype = torch.bfloat16):
    """``(k, v)`` [B,H,length,D] in ``dtype`` (bf16: exactly what the cache holds; fp16: rounded below its normal numbers, and
    61440 where the cache holds more than its 65504): the first
    ``lens[b]`` tokens of every sequence, zeros behind them and where the table names no page.  ``length`` defaults to the
    tokens the table has place for.  Any window of the table's columns reads those pages (with lengths that count from there)."""
    return _native.host().paged_gather(cache, page_table, lens, length, dtype)


def paged_cache_copy(cache: PagedCache, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` (int32 [n] on the cache's device).  Pairs with a number that is no page are left out; a
    destination named more than once takes the last one's page.  No page may be both a source and a destination."""
    _native.host().paged_copy(cache, src, dst)


def paged_cache_fork(cache: PagedCache, page_table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor,
                     new_pages: torch.Tensor):
    """``(page_table, lens)`` of n new sequences that continue ``parents`` (int32 [n], repeats allowed): full pages are
    shared, a last page that is not full is copied to ``new_pages[i]`` (int32 [n], free pages), which then stands in
    the new row.  Where ``new_pages[i]`` is no page (-1, say) the child keeps its parent's last page: for one child of each
    parent that is not itself continued.  Entries behind the last page are -1; a parent that is no sequence gives an empty one."""
    return _native.host().paged_fork(cache, page_table, lens, parents, new_pages)


def paged_cache_compact(cache: PagedCache, page_table: torch.Tensor, lens: torch.Tensor):
    """Moves the pages that the sequences use to the front of the pool: ``(page_table, used)``, the table with the pages'
    new numbers (-1 behind each sequence's last page) and their number, int32 [1].  Pages from ``used`` on move to the free ones
    below it, the lowest to the lowest; shared pages stay shared.  Every sequence that is to live must be in the table: a page
    that only other tables, or entries behind ``lens``, name is free.  ``page_table`` itself is not changed."""
    return _native.host().paged_compact(cache, page_table, lens)


def paged_cache_free_pages(cache: PagedCache, page_table: torch.Tensor, lens: torch.Tensor):
    """``(pages, count)``: the pages that no sequence uses, int32 [num_pages] in rising order with -1 behind the last, and
    how many they are, int32 [1].  A sequence is freed by setting its length to 0."""
    return _native.host().paged_free_pages(cache, page_table, lens)


def sparse_attention_decode_paged(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lens: torch.Tensor,
                                  mask: Optional[torch.Tensor] = None, mask_metadata: Optional[MaskMetadata] = None, *,
                                  counts: Optional[torch.Tensor] = None, window: Optional[int] = None, return_lse: bool = False):
    """:func:`sparseattention_amd.sparse_attention_decode` over a paged cache: ``q`` [B,Hq,Sq,D] (bf16 or fp16, 1 <= Sq <= 32) against the
    first ``lens[b]`` tokens of every sequence, the call's own among them.  Hq is a multiple of the cache's H: query heads
    ``h * Hq / H`` and following read K/V head ``h``.  Returns ``o`` like q or, with ``return_lse``, ``(o, lse)`` as there.

    Without a mask row ``i`` attends to keys ``0 .. lens[b] - n + i``, n the number of rows: causal, the rows being the last tokens;
    with ``window`` to the last ``window`` of these.  ``counts`` (int32 [B]): n differs, rows ``counts[b]`` and following of sequence ``b``
    are padding and give 0 (``lse`` -inf).
    ``mask``: bool broadcastable to [B,H,Sq,Sk], H the K/V heads, Sk whole pages, True = attend; it replaces causality, and keys from
    ``lens[b]`` on are left out whatever it says.  ``mask_metadata``: ``compute_mask_kernel(mask, Sq, page_size)``, with which no mask is
    needed; only the pages it lists are read.

    Probabilities and values meet in q's type, sums are float32; with fp16 queries the values are those that
    ``paged_cache_gather(..., dtype=torch.float16)`` gives."""
    return _native.host().decode_paged(q, cache, page_table, lens, mask, mask_metadata, counts, window, return_lse)
