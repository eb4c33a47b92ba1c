"""Calls of the paged cache at the edges of what it documents, on the CPU:
nothing here launches a kernel."""

import pytest
import torch

from layer_streaming import PagedKVCache, _hip


def small_cache(**changes):
    sizes = dict(num_pages=4, max_sequences=3, max_length=20, layer_count=1, num_kv_heads=2,
                 head_dim=64, page_size=8, device="cpu")
    return PagedKVCache(**dict(sizes, **changes))


def test_extend_of_no_rows_changes_nothing():
    # a step of a serving loop with no live sequence
    cache = small_cache()
    row = cache.add()
    cache.extend([row], 3)
    for rows in ([], (), torch.empty(0, dtype=torch.int64)):
        cache.extend(rows)
        cache.extend(rows, 5)
    with pytest.raises(ValueError):
        cache.extend([], 0)
    assert cache.length(row) == 3 and cache.free_pages == 3
    assert cache.lengths.tolist() == [3, 0, 0] and cache.page_table[0].tolist() == [0, -1, -1]


@pytest.mark.parametrize("max_length,page_size", [(500, 1024), (20, 8), (1000, 1024)])
def test_the_caches_workspace_serves_every_limit(max_length, page_size):
    # attend takes limits of up to what a table row holds, which is more than
    # max_length where that ends inside a page
    cache = small_cache(max_length=max_length, page_size=page_size)
    capacity = cache.max_pages * page_size
    assert capacity > max_length
    held = cache._attention_workspace(3, 8).numel()
    for limit in (1, max_length, capacity):
        assert held >= _hip.paged_attention_workspace_bytes(3, 8, 2, 64, limit)
