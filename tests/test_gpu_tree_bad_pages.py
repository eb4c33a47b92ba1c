"""Drafted trees' attention beside pages outside the pool: their positions are
left out as if masked, and nothing else is."""

import math

import pytest
import torch

from layer_streaming import _hip
from paged_cases import Pool
from tree_cases import Step, attention

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("past,nodes", [(100, 5), (100, 40), (1900, 9), (2500, 9)])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(8, 2, 128, 8), (6, 2, 64, 16)])
def test_infinities_on_the_good_pages_of_a_block(gpu_device, past, nodes, value, q_heads,
                                                 kv_heads, dim, page):
    # position 33 is on a page outside the pool, 55 in the same 32 positions
    print("bad page", past, nodes, value, dim, flush=True)
    pool = Pool([past + nodes, 70], kv_heads, dim, page, seed=past)
    step = Step([nodes, 3], [0, 1], q_heads, dim, seed=nodes, spare=1)
    good_page = int(pool.table[0, 55 // page])
    pool.table[0, 33 // page] = pool.k.shape[0]
    pool.v[good_page, :, 55 % page, 4] = value
    limit = pool.table.shape[1] * page
    q, starts, masks, rows = step.tensors(gpu_device)
    size = _hip.paged_tree_attention_workspace_bytes(2, nodes, q_heads, kv_heads, dim, limit)
    out = torch.full_like(q, 7.0)
    error = torch.zeros(1, dtype=I32, device=gpu_device)
    _hip.paged_tree_attention(
        q, starts, masks, pool.k.to(gpu_device), pool.v.to(gpu_device),
        pool.table.to(gpu_device), pool.lengths.to(gpu_device), out,
        torch.full((size,), 0xFF, dtype=torch.uint8, device=gpu_device), dim ** -0.5, rows=rows,
        max_tree=nodes, error_flag=error)
    out = out.cpu()
    assert int(error.item()) == _hip.PAGED_ERANGE
    hit = out[:nodes, :, 4].float()
    assert bool((hit.isnan() if math.isnan(value) else hit == value).all()), hit
    # the other dims, the other tree, and the row behind them
    pool.v[good_page, :, 55 % page, 4] = 0
    for b in range(2):
        length = int(pool.lengths[b])
        k, v, good = pool.rows_of(b, length)
        for t in range(step.starts[b], step.starts[b + 1]):
            seen = step.seen(b, t - step.starts[b], length, good)
            ref, tol = attention(step.q[t], k, v, seen, dim ** -0.5)
            off = (out[t].double() - ref).abs()
            if b == 0:
                off[:, 4] = 0
            assert bool((off <= tol).all()), (b, t)
    assert bool((out[-1] == 7).all())
