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


@pytest.fixture
def copies(monkeypatch):
    """copy_pages on the CPU up to its launch: (planes, plane bytes, pages,
    page bytes) of each."""

    calls = []
    monkeypatch.setattr(_hip, "_gpu_of", lambda name, tensor: tensor.device)
    monkeypatch.setattr(
        _hip, "_call_on", lambda index, stream, name, at, *sizes: calls.append(sizes[:4]))
    return calls


PAIRS = torch.tensor([[0, 1]], dtype=torch.int32)


def test_copy_pages_refuses_one_layers_pools(copies):
    # [2, pages, kv_heads, page_size, dim] is no [layers, 2, pages, ...]: its
    # KV heads would pass for pages.  With two pages it looks like two layers
    for pages in (4, 3, 2):
        cache = small_cache(num_pages=pages)
        with pytest.raises(ValueError, match="flatten"):
            _hip.copy_pages(cache.buffer[0], PAIRS)
    with pytest.raises(ValueError):
        _hip.copy_pages(torch.zeros(2, 3, 4, 2, 8, 64), PAIRS)
    assert not copies


def test_copy_pages_reads_planes(copies):
    cache = small_cache(layer_count=3)
    page = 2 * 8 * 64 * 2
    _hip.copy_pages(cache.buffer, PAIRS)
    _hip.copy_pages(cache.buffer.flatten(0, 1).flatten(2), PAIRS)
    _hip.copy_pages(cache.buffer[0].flatten(2), PAIRS)
    _hip.copy_pages(torch.zeros(3, 2, 4, 16, 64, dtype=torch.bfloat16), PAIRS)
    _hip.copy_pages(cache.k_pages(1)[None].flatten(2), PAIRS)
    assert copies == [(6, 4 * page, 4, page)] * 2 + [(2, 4 * page, 4, page)] + [
        (6, 4 * 2048, 4, 2048), (1, 4 * page, 4, page)]


@pytest.mark.parametrize("head_dim", [0, 8, 72, 1040, -64])
def test_head_sizes_that_no_operator_takes_are_refused(head_dim):
    with pytest.raises(ValueError):
        small_cache(head_dim=head_dim)


def test_attend_names_head_sizes_it_does_not_take():
    # append and the copies take them: the refusal is attend's
    cache = small_cache(head_dim=96)
    q = torch.zeros(1, 4, 96, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="64 or 128"):
        cache.attend(0, q, torch.zeros_like(q))


def test_the_caches_workspace_of_the_longest_sequences():
    # the last page of the longest row ends past what attention takes
    longest = 2 ** 31 - 1 - 64
    cache = small_cache(max_length=longest, page_size=1024, max_sequences=1)
    held = cache._attention_workspace(3, 8).numel()
    assert held >= _hip.paged_attention_workspace_bytes(3, 8, 2, 64, longest)
