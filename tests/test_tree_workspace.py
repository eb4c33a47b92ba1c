"""The size of the drafted trees' workspace serves every smaller call, on the
CPU."""

import ctypes

import pytest

from layer_streaming import _hip

SHAPES = [(32, 8, 128), (40, 8, 128), (28, 4, 128), (7, 1, 64), (16, 1, 128), (8, 1, 128),
          (64, 8, 128), (48, 3, 64), (14, 14, 64), (12, 4, 64), (30, 2, 128)]


@pytest.mark.parametrize("q_heads,kv_heads,dim", SHAPES)
def test_smaller_calls_never_need_more(q_heads, kv_heads, dim):
    size = _hip.paged_tree_attention_workspace_bytes
    for limit in (500, 3000, 32768, 65536):
        for trees in (1, 2, 24, 100, 300):
            needs = [size(trees, nodes, q_heads, kv_heads, dim, limit)
                     for nodes in range(1, 65)]
            assert needs == sorted(needs), (trees, limit)
    for nodes in (1, 17, 36, 51, 64):
        needs = [size(trees, nodes, q_heads, kv_heads, dim, 32768) for trees in range(1, 400, 3)]
        assert needs == sorted(needs), nodes
        needs = [size(3, nodes, q_heads, kv_heads, dim, limit) for limit in range(1, 9000, 37)]
        assert needs == sorted(needs), nodes


@pytest.mark.parametrize("q_heads,kv_heads,dim,largest,smaller", [
    (8, 1, 128, 33, 32), (64, 8, 128, 33, 32), (40, 8, 128, 64, 51), (16, 1, 128, 64, 48)])
def test_the_entry_point_takes_a_larger_calls_workspace(q_heads, kv_heads, dim, largest,
                                                        smaller):
    # refused for its error word's alignment before anything is launched; the
    # size is looked at behind that
    lib = _hip.load()
    limit, page = 32768, 64
    given = _hip.paged_tree_attention_workspace_bytes(2, largest, q_heads, kv_heads, dim, limit)
    need = _hip.paged_tree_attention_workspace_bytes(2, smaller, q_heads, kv_heads, dim, limit)
    assert need <= given
    stride = kv_heads * page * dim
    args = [16, q_heads * dim, dim, 2 * smaller, 16, 16, 2, smaller, 16, 16, stride, page * dim,
            2000, page, 16, limit // page, 4, 16, 16, limit, q_heads, kv_heads, dim,
            ctypes.c_float(0.1), 16, q_heads * dim, dim, 16]
    fn = lib.cascade_paged_tree_attention_bf16
    assert fn(*args, given, 18, None) == 1002
    assert fn(*args, 4096, 16, None) == 1004
