"""Caches over tensors with a size of 0 are refused by every operator, on the host before anything is computed from their sizes (runs without
a GPU)."""
import pytest
import torch

import sparseattention_amd as sa


@pytest.mark.parametrize("pages,H,per", [(4, 0, 2), (0, 2, 2), (4, 2, 0), (0, 0, 0)])
def test_caches_without_pages_heads_or_tokens(pages, H, per):
    cache = sa.PagedCache(*(torch.zeros(pages, H, per, 2048, dtype=torch.uint8) for _ in range(2)), *(torch.zeros(pages, H, per) for _ in range(2)), 64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, H, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: sa.sparse_attention_decode_paged(x.new_zeros(1, 2, 1, 64), cache, table, lens),
                 lambda: sa.paged_cache_append(cache, x, x, table, lens), lambda: sa.paged_cache_gather(cache, table, lens),
                 lambda: sa.paged_cache_copy(cache, lens, lens), lambda: sa.paged_cache_fork(cache, table, lens, lens, lens),
                 lambda: sa.paged_cache_compact(cache, table, lens), lambda: sa.paged_cache_free_pages(cache, table, lens)):
        with pytest.raises(ValueError, match="cache"):
            call()
