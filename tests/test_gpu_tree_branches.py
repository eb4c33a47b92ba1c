"""Drafted trees' attention where its rarer paths are taken: split batches of
more than 64 trees, scores that climb past the running reference, scales of any
sign."""

import pytest
import torch

from layer_streaming import _hip
from paged_cases import Pool
from tree_cases import Step, attention

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


def check(pool, step, out, scale):
    for b, row in enumerate(step.rows):
        length = int(pool.lengths[row])
        k, v, good = pool.rows_of(row, length)
        for t in range(step.starts[b], step.starts[b + 1]):
            seen = step.seen(b, t - step.starts[b], length, good)
            # (a negative scale is a positive one of -q)
            ref, tol = attention(step.q[t] if scale >= 0 else -step.q[t], k, v, seen, abs(scale))
            off = (out[t].double() - ref).abs()
            assert bool((off <= tol).all()), (b, t, float((off - tol).max()))
    assert bool((out[step.starts[-1]:] == 7).all())


@pytest.mark.parametrize("trees,q_heads,kv_heads,dim", [(65, 8, 2, 128), (150, 6, 2, 64),
                                                        (256, 4, 1, 128)])
def test_split_batches_of_more_than_64_trees(gpu_device, trees, q_heads, kv_heads, dim):
    # the long ones lie past the 64th, and one among the first
    print("split batch", trees, dim, flush=True)
    long = {3: 2100, 64: 3000, 66: 2500, trees - 1: 4000, trees // 2 + 20: 900}
    past = [long.get(i, i * 37 % 90) for i in range(trees)]
    sizes = [1 + i * 5 % 7 for i in range(trees)]
    pool = Pool([p + n for p, n in zip(past, sizes)], kv_heads, dim, 16, seed=trees)
    step = Step(sizes, range(trees), q_heads, dim, seed=trees)
    out = attend(pool, step, gpu_device, 7, dim ** -0.5)
    check(pool, step, out, dim ** -0.5)


def climbing(pool, step, row, length, rate, until):
    """Keys along the queries, whose scores climb by ``rate`` powers of two every
    96 positions up to ``until`` and fall behind it; the values' sizes fall as the
    weights climb, so that all of them count."""

    dim, page = step.q.shape[2], pool.k.shape[2]
    step.q[..., 0] = 2
    for p in range(length):
        stage = min(p, max(0, 2 * until - p)) / 96
        at = int(pool.table[row, p // page]), p % page
        pool.k[at[0], :, at[1], 0] = stage * rate * 0.6931 / (2 * dim ** -0.5)
        scale = 2.0 ** -min(60.0, stage * rate)
        pool.v[at[0], :, at[1]] = (pool.v[at[0], :, at[1]].float() * scale).to(torch.bfloat16)


@pytest.mark.parametrize("rate", [3.0, 9.0, 30.0])
@pytest.mark.parametrize("past,nodes,q_heads,kv_heads,dim", [
    (450, 9, 8, 2, 128), (400, 60, 8, 2, 64), (3000, 5, 8, 2, 128), (3000, 33, 16, 1, 128),
    (5000, 9, 8, 2, 64)])
def test_scores_that_climb(gpu_device, past, nodes, q_heads, kv_heads, dim, rate):
    # by 2^8 and more above the reference of the exponents, again and again
    print("climb", past, nodes, dim, rate, flush=True)
    pool = Pool([past + nodes], kv_heads, dim, 16, seed=past)
    step = Step([nodes], [0], q_heads, dim, seed=nodes)
    climbing(pool, step, 0, past + nodes, rate, past * 2 // 3)
    out = attend(pool, step, gpu_device, nodes, dim ** -0.5)
    check(pool, step, out, dim ** -0.5)


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.09, -1.0, 1e-30, 1e-40, 0.5])
@pytest.mark.parametrize("past,nodes", [(70, 9), (2500, 20)])
def test_scales_of_any_sign(gpu_device, past, nodes, scale):
    print("scale", past, nodes, scale, flush=True)
    pool = Pool([past + nodes, 3], 2, 64, 16, seed=past)
    step = Step([nodes, 3], [0, 1], 8, 64, seed=nodes)
    out = attend(pool, step, gpu_device, nodes, scale)
    check(pool, step, out, scale)


@pytest.mark.parametrize("q_heads,kv_heads,dim,largest,nodes", [
    (40, 8, 128, 64, 51), (28, 4, 128, 64, 36), (7, 1, 64, 64, 36), (16, 1, 128, 64, 48)])
def test_a_workspace_sized_for_larger_trees(gpu_device, q_heads, kv_heads, dim, largest, nodes):
    # fewer nodes take fewer workgroups a run, and so more runs
    print("workspace", q_heads, kv_heads, largest, nodes, flush=True)
    limit, page = 32768, 64
    pool = Pool([2900 + nodes], kv_heads, dim, page, seed=nodes, width=limit // page)
    step = Step([nodes], [0], q_heads, dim, seed=largest)
    q, starts, masks, rows = step.tensors(gpu_device)
    size = _hip.paged_tree_attention_workspace_bytes(1, largest, q_heads, kv_heads, dim, limit)
    # (what lies behind it stays)
    space = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=gpu_device)
    out = torch.full_like(q, 7.0)
    _hip.paged_tree_attention(
        q, starts, masks, pool.k.to(gpu_device), pool.v.to(gpu_device),
        pool.table.to(gpu_device), pool.lengths.to(gpu_device), out, space[:size], dim ** -0.5,
        rows=rows, max_tree=nodes)
    check(pool, step, out.cpu(), dim ** -0.5)
    assert bool((space[size:] == 0xA5).all())
