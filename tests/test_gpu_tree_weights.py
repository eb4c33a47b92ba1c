"""What weights of the drafted trees' attention keep: all bits of fp32 in the
product with V, and infinities of V under any weight."""

import math

import pytest
import torch

from layer_streaming import _hip
from paged_cases import Pool
from tree_cases import Step

pytestmark = pytest.mark.gpu

I32 = torch.int32


def attend(pool, step, device, max_tree, scale):
    limit = pool.table.shape[1] * pool.k.shape[2]
    q, starts, masks, rows = step.tensors(device)
    size = _hip.paged_tree_attention_workspace_bytes(
        len(step.rows), max_tree, q.shape[1], pool.k.shape[1], q.shape[2], limit)
    out = torch.full_like(q, 7.0)
    error = torch.zeros(1, dtype=I32, device=device)
    _hip.paged_tree_attention(
        q, starts, masks, pool.k.to(device), pool.v.to(device), pool.table.to(device),
        pool.lengths.to(device), out, torch.full((size,), 0xFF, dtype=torch.uint8, device=device),
        scale, rows=rows, max_tree=max_tree, error_flag=error)
    torch.cuda.synchronize(device)
    assert int(error.item()) == 0
    return out.cpu()


def place(pool, position):
    page = pool.k.shape[2]
    return int(pool.table[0, position // page]), position % page


def scores(pool, step, length):
    """Scores that one product makes: q is 1 in the first dim and 0 elsewhere, K
    holds the scores there.  Returns them, [kv_heads, length]."""

    pool.k[:] = 0
    step.q[:] = 0
    step.q[..., 0] = 1
    g = torch.Generator().manual_seed(length)
    dim = step.q.shape[2]
    s = (torch.rand(pool.k.shape[1], length, generator=g) * 4 - 2) * dim ** 0.5
    s = s.to(torch.bfloat16)
    for p in range(length):
        page, slot = place(pool, p)
        pool.k[page, :, slot, 0] = s[:, p]
    return s.double()


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(8, 4, 128), (8, 4, 64), (64, 4, 128)])
@pytest.mark.parametrize("past,nodes", [(40, 5), (40, 60), (2500, 9)])
def test_the_product_with_v_has_all_bits_of_the_weights(gpu_device, past, nodes, q_heads,
                                                        kv_heads, dim):
    """Values chosen so that sum w V nearly cancels show what the weights lost.

    Bound, relative to sum w |V|: the scores are exact; their scaling to powers
    of two is off by 2^-23 of up to 2.9 and the argument by half a step of up to
    5.8, together 2^-21.4 times ln 2; exp2 by 2^-23; a group's own reference by
    2^-24 of 2.9; sums of the 16 positions that count, cut at 2^-23 of what is
    summed, round three times a product and twice in the joins.  Less than
    2^-19 in all, where weights of 16 bits are off by up to 2^-16."""

    print("weights", past, nodes, q_heads, dim, flush=True)
    length = past + nodes
    pool = Pool([length], kv_heads, dim, 16, seed=past)
    step = Step([nodes], [0], q_heads, dim, seed=nodes, spare=0)
    step.masks = [(1 << 64) - 1] * nodes  # every node sees everything
    s = scores(pool, step, length) * dim ** -0.5
    w = torch.softmax(s, -1)
    pool.v[:] = 0
    g = torch.Generator().manual_seed(past + nodes)
    at = torch.randperm(length, generator=g)[:16].tolist()
    total = torch.zeros(kv_heads, dim, dtype=torch.float64)
    size = torch.zeros_like(total)
    for i, p in enumerate(at):
        if i < 12:
            v = torch.randn(kv_heads, dim, generator=g, dtype=torch.float64)
        else:
            v = -total / w[:, p, None]
        v = v.to(torch.bfloat16)
        page, slot = place(pool, p)
        pool.v[page, :, slot] = v
        total += w[:, p, None] * v.double()
        size += w[:, p, None] * v.double().abs()
    assert bool((total.abs() < 2.0 ** -22 * size).all())
    out = attend(pool, step, gpu_device, nodes, dim ** -0.5).double()
    group = q_heads // kv_heads
    total, size = (x.repeat_interleave(group, 0) for x in (total, size))
    off = (out - total).abs() / size
    assert bool((off < 2.0 ** -19).all()), math.log2(float(off.max()))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("under", [0.0, -1.0, -300.0])
@pytest.mark.parametrize("past,nodes", [(100, 5), (2500, 40)])
def test_an_infinity_before_the_tree(gpu_device, past, nodes, under, value):
    # under the largest weight, which is a power of two, an ordinary one and one
    # that fp32 does not hold; other dims stay as they are without it
    print("infinity", past, nodes, under, value, flush=True)
    dim, length = 128, past + nodes
    pool = Pool([length], 2, dim, 16, seed=past)
    step = Step([nodes], [0], 8, dim, seed=nodes, spare=0)
    scores(pool, step, length)
    page, slot = place(pool, 37)
    pool.k[page, :, slot, 0] = (3.0 + under) * dim ** 0.5
    clean = attend(pool, step, gpu_device, nodes, dim ** -0.5)
    pool.v[page, :, slot, 3] = value
    pool.v[page, :, slot, dim - 2] = value
    out = attend(pool, step, gpu_device, nodes, dim ** -0.5)
    hit = out[:, :, [3, dim - 2]].float()
    assert bool((hit.isnan() if math.isnan(value) else hit == value).all())
    keep = [d for d in range(dim) if d not in (3, dim - 2)]
    assert torch.equal(out[:, :, keep], clean[:, :, keep])
    assert bool(clean.isfinite().all())


@pytest.mark.parametrize("value", [3e35, -6e35])
@pytest.mark.parametrize("past,nodes", [(100, 5), (2500, 40)])
def test_large_values_under_no_weight(gpu_device, past, nodes, value):
    # finite, under a weight that fp32 does not hold, in a run of their own: they
    # are worth nothing.  Two of 6e35, each times 2^8 at most, are 3.1e38: sums that
    # are divided at the end stay in fp32's range, as the operator asks.
    print("large", past, nodes, value, flush=True)
    dim, length = 128, past + nodes
    pool = Pool([length], 2, dim, 16, seed=past)
    step = Step([nodes], [0], 8, dim, seed=nodes, spare=0)
    scores(pool, step, length)
    for p in range(past // 2):
        page, slot = place(pool, p)
        pool.k[page, :, slot, 0] = -300 * dim ** 0.5
    clean = attend(pool, step, gpu_device, nodes, dim ** -0.5)
    for p in (3, 37):
        page, slot = place(pool, p)
        pool.v[page, :, slot, 3:9] = value
    out = attend(pool, step, gpu_device, nodes, dim ** -0.5)
    assert torch.equal(out, clean) and bool(clean.isfinite().all())
