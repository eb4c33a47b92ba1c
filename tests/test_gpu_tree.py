"""Drafted trees against their plain forms: attention of the nodes in 64 bits,
acceptance with the move of K and V rows exactly, the append at rope rows of
its own; and steps of them together."""

import math
import random

import pytest
import torch

from layer_streaming import PagedKVCache, _hip, tree_masks
from paged_cases import Pool, normal, rotated
from tree_cases import Step, attention, random_parents, walk

pytestmark = pytest.mark.gpu

I32, I64 = torch.int32, torch.int64


def flag(device):
    return torch.zeros(1, dtype=I32, device=device)


def workspace(step, pool, max_tree, limit, device):
    size = _hip.paged_tree_attention_workspace_bytes(
        max(1, len(step.rows)), max_tree, step.q.shape[1], pool.k.shape[1], pool.k.shape[3],
        limit)
    return torch.full((size,), 0xFF, dtype=torch.uint8, device=device)


def attend(pool, step, device, max_tree=64, limit=None, out=None, ws=None, error=None,
           rows=True):
    """Run the operator; returns (out on the CPU, flag)."""

    limit = pool.table.shape[1] * pool.k.shape[2] if limit is None else limit
    q, starts, masks, row_of = step.tensors(device)
    out = torch.full_like(q, 7.0) if out is None else out
    error = flag(device) if error is None else error
    ws = workspace(step, pool, max_tree, limit, device) if ws is None else ws
    got = _hip.paged_tree_attention(
        q, starts, masks, pool.k.to(device), pool.v.to(device), pool.table.to(device),
        pool.lengths.to(device), out, ws, q.shape[2] ** -0.5, rows=row_of if rows else None,
        max_tree=max_tree, max_length=limit, error_flag=error)
    assert got is out
    torch.cuda.synchronize(device)
    return out.cpu(), int(error.item())


def check(pool, step, out, left_out=()):
    live = torch.zeros(out.shape[0], dtype=torch.bool)
    for b, row in enumerate(step.rows):
        first, end = step.starts[b], step.starts[b + 1]
        if row < 0 or b in left_out:
            continue
        length = int(pool.lengths[row])
        k, v, good = pool.rows_of(row, length)
        for t in range(first, end):
            live[t] = True
            ref, tol = attention(step.q[t], k, v, step.seen(b, t - first, length, good),
                                 step.q.shape[2] ** -0.5)
            off = (out[t].double() - ref).abs()
            assert bool((off <= tol).all()), (b, row, t - first, length,
                                              float((off - tol).max()), float(off.max()))
    assert bool((out[~live] == 7).all()), "a row of no tree was written"


SHAPES = [(32, 8, 128), (5, 5, 64), (16, 1, 128), (12, 4, 64), (6, 2, 128), (32, 2, 64),
          (9, 1, 64)]
# (past, nodes)
MIXED = [(0, 1), (0, 64), (1, 2), (31, 1), (7, 16), (30, 5), (32, 17), (200, 33), (0, 0),
         (500, 63), (129, 3), (1000, 8), (13, 0)]


@pytest.mark.parametrize("q_heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("page_size", [8, 16, 64, 256])
def test_trees_of_all_sizes(gpu_device, q_heads, kv_heads, dim, page_size):
    print("trees", q_heads, kv_heads, dim, page_size, flush=True)
    pool = Pool([p + n for p, n in MIXED], kv_heads, dim, page_size, seed=page_size + q_heads)
    rows = list(range(len(MIXED)))
    random.Random(page_size).shuffle(rows)
    step = Step([MIXED[r][1] for r in rows], rows, q_heads, dim, seed=q_heads)
    out, error = attend(pool, step, gpu_device)
    check(pool, step, out)
    assert error == 0


@pytest.mark.parametrize("max_tree", [1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 24, 31, 32, 33, 48, 63, 64])
def test_widths(gpu_device, max_tree):
    # trees of up to the width that the call names, arbitrary masks
    print("width", max_tree, flush=True)
    sizes = [max_tree, 1, max(1, max_tree // 2), 0, max(1, max_tree - 1)]
    past = [70, 3, 600, 5, 33]
    for q_heads, kv_heads, dim in ((8, 2, 128), (6, 2, 64)):
        pool = Pool([p + n for p, n in zip(past, sizes)], kv_heads, dim, 16, seed=max_tree)
        step = Step(sizes, range(5), q_heads, dim, seed=max_tree, masks="any")
        out, error = attend(pool, step, gpu_device, max_tree=max_tree, rows=False)
        check(pool, step, out)
        assert error == 0


@pytest.mark.parametrize("trees,past,nodes,page_size", [
    (1, 0, 1, 8), (1, 40, 4, 16), (1, 9000, 16, 64), (2, 5000, 64, 16), (150, 70, 5, 8),
    (3, 20001, 9, 128), (1, 33000, 33, 64), (1030, 20, 2, 8), (300, 700, 3, 32)])
def test_batches(gpu_device, trees, past, nodes, page_size):
    print("batch", trees, past, nodes, page_size, flush=True)
    sizes = [max(1, nodes - i % 3) for i in range(trees)]
    lengths = [max(0, past - 37 * i) + n for i, n in enumerate(sizes)]
    pool = Pool(lengths, 2, 128, page_size, seed=trees)
    step = Step(sizes, range(trees), 8, 128, seed=past)
    out, error = attend(pool, step, gpu_device, max_tree=nodes)
    check(pool, step, out)
    assert error == 0


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(16, 4, 128), (16, 4, 64)])
@pytest.mark.parametrize("trees", [2, 70])
@pytest.mark.parametrize("width", [4, 8, 16, 30, 60])
def test_short_trees(gpu_device, trees, width, q_heads, kv_heads, dim):
    # one workgroup a tree and KV head, of two widths: fewer than the device has
    # CUs, and more
    print("short", trees, width, dim, flush=True)
    sizes = [width if i == 0 else 1 + i * 7 % min(width, 12) for i in range(trees)]
    past = [i * 61 % 440 for i in range(trees)]
    pool = Pool([p + n for p, n in zip(past, sizes)], kv_heads, dim, 16, seed=width)
    step = Step(sizes, range(trees), q_heads, dim, seed=trees)
    out, error = attend(pool, step, gpu_device, max_tree=width)
    check(pool, step, out)
    assert error == 0


@pytest.mark.parametrize("trees", [64, 30, 12])
@pytest.mark.parametrize("dim,width", [(128, 3), (64, 9), (128, 20)])
def test_long_trees_whole_and_split(gpu_device, trees, dim, width):
    # 512 workgroups take sequences of up to 2048 positions whole, 240 split them
    print("whole", trees, dim, width, flush=True)
    sizes = [width if i < 2 else 1 + i % 2 for i in range(trees)]
    past = [2047 - width, 1000] + [i * 331 % 900 for i in range(2, trees)]
    pool = Pool([p + n for p, n in zip(past, sizes)], 8, dim, 16, seed=width)
    step = Step(sizes, range(trees), 16, dim, seed=trees)
    out, error = attend(pool, step, gpu_device, max_tree=width)
    check(pool, step, out)
    assert error == 0


def test_a_mask_of_nothing(gpu_device):
    # no past and an empty mask: zeros; with a past: the past alone
    pool = Pool([4, 40], 2, 128, 8, seed=1)
    step = Step([4, 4], [0, 1], 8, 128, seed=2)
    step.masks[1] = step.masks[5] = 0
    step.masks[2] = 0xF0  # bits past the tree
    out, error = attend(pool, step, gpu_device)
    check(pool, step, out)
    assert bool((out[1] == 0).all()) and bool((out[2] == 0).all()) and error == 0


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("q_heads,kv_heads,dim,past", [(8, 2, 128, 30), (8, 2, 64, 0),
                                                       (32, 8, 128, 700), (16, 1, 64, 1500)])
def test_values_that_a_node_does_not_see(gpu_device, value, q_heads, kv_heads, dim, past):
    # two chains from the root: one of them holds values that are no numbers
    nodes = 40
    pool = Pool([past + nodes], kv_heads, dim, 8, seed=3)
    step = Step([nodes], [0], q_heads, dim, seed=4)
    parents = [-1, 0, 0] + [i - 2 for i in range(3, nodes)]
    step.masks[:nodes] = [m & (1 << 64) - 1 for m in tree_masks(parents)[0]]

    def at(position):
        return int(pool.table[0, position // 8]), position % 8

    bad = 11
    page, slot = at(past + bad)
    pool.v[page, :, slot, 5] = value
    pool.v[page, :, slot, dim - 1] = value
    last, last_slot = at(past + nodes - 1)  # nobody but itself sees it
    pool.k[last, :, last_slot] = value
    out, _ = attend(pool, step, gpu_device)
    sees = torch.tensor([bool(m >> bad & 1) for m in step.masks[:nodes]])
    sees[nodes - 1] = False  # (looked at below)
    for t in range(nodes - 1):
        row = out[t].float()
        want = row[:, [5, dim - 1]]
        if sees[t]:
            good = want.isnan() if math.isnan(value) else want == value
            assert bool(good.all()), (t, want)
            row[:, [5, dim - 1]] = 0
        assert bool(row.isfinite().all()), t
    assert not bool(out[nodes - 1].isfinite().all()) or not math.isnan(value)
    # with finite values in their places, the nodes that saw none of it agree
    pool.v[page, :, slot] = 1.0
    pool.k[last, :, last_slot] = 1.0
    clean, _ = attend(pool, step, gpu_device)
    check(pool, step, clean)
    for t in range(nodes - 1):
        if not sees[t]:
            assert bool((clean[t] == out[t]).all()), t


def test_an_infinite_value_next_to_its_negative(gpu_device):
    # seen together they have no sum, apart they keep their sign
    pool = Pool([6], 1, 64, 8, seed=5)
    page = int(pool.table[0, 0])
    pool.v[page, 0, 2, 0] = math.inf
    pool.v[page, 0, 3, 0] = -math.inf
    step = Step([6], [0], 4, 64, seed=6)
    step.masks[:6] = [0b000001, 0b000011, 0b000101, 0b001001, 0b001101, 0b110001]
    out, _ = attend(pool, step, gpu_device)
    first = out[:6, :, 0].float()
    assert bool(first[[0, 1, 5]].isfinite().all())
    assert bool((first[2] == math.inf).all()) and bool((first[3] == -math.inf).all())
    assert bool(first[4].isnan().all()) and bool(out[:6, :, 1:].isfinite().all())


def test_rows_padding_and_strides(gpu_device):
    # trees in another order, padding, q and out as views of wider rows, pools
    # as views of a larger buffer
    pool = Pool([300, 12, 64, 3, 1000], 4, 64, 16, seed=1, width=80)
    step = Step([7, 3, 9, 0, 12, 1], [4, -1, 0, 2, 1, 3], 12, 64, seed=8, spare=5)
    fused = torch.zeros(step.q.shape[0], 24, 64, dtype=torch.bfloat16)
    fused[:, 3:15] = step.q
    fused = fused.to(gpu_device)
    wide = torch.full((step.q.shape[0], 20, 64), 7.0, dtype=torch.bfloat16, device=gpu_device)
    buffer = torch.stack((pool.k, pool.v)).to(gpu_device)
    both = torch.stack((buffer, buffer)).transpose(1, 2).contiguous()
    _, starts, masks, rows = step.tensors(gpu_device)
    error = flag(gpu_device)
    _hip.paged_tree_attention(
        fused[:, 3:15], starts, masks, both[1, :, 0], both[1, :, 1],
        pool.table.to(gpu_device), pool.lengths.to(gpu_device), wide[:, 4:16],
        workspace(step, pool, 12, 1280, gpu_device), 64 ** -0.5, rows=rows, max_tree=12,
        error_flag=error)
    check(pool, step, wide[:, 4:16].cpu())
    assert bool((wide[:, :4] == 7).all()) and bool((wide[:, 16:] == 7).all())
    assert int(error.item()) == 0


@pytest.mark.parametrize("past", [20, 900])
def test_what_is_out_of_range_is_flagged(gpu_device, past):
    sizes = [3, 4, 2, 5]
    pool = Pool([past + n for n in sizes], 2, 128, 16, seed=2)

    def run(change, left_out, limit=None, max_tree=8):
        step = Step(sizes, range(4), 8, 128, seed=7)
        lengths = pool.lengths.clone()
        change(step, pool)
        out, error = attend(pool, step, gpu_device, max_tree=max_tree, limit=limit)
        assert error == _hip.PAGED_ERANGE
        check(pool, step, out, left_out)
        pool.lengths = lengths

    run(lambda s, p: s.rows.__setitem__(1, 4), [1])
    run(lambda s, p: s.rows.__setitem__(1, 1 << 30), [1])
    run(lambda s, p: p.lengths.__setitem__(2, 1), [2])  # below its nodes
    run(lambda s, p: p.lengths.__setitem__(2, -5), [2])
    run(lambda s, p: None, [3], limit=past + 4)
    run(lambda s, p: None, [3], max_tree=4)
    run(lambda s, p: s.starts.__setitem__(4, 100), [3])
    run(lambda s, p: s.starts.__setitem__(0, -1), [0])
    run(lambda s, p: s.starts.__setitem__(1, 15), [0, 1])  # too many, and backwards
    # a page outside the pool: its positions take no part
    for page in (-1, pool.k.shape[0], 1 << 30):
        good = pool.table.clone()
        pool.table[0, 0] = page
        step = Step(sizes, range(4), 8, 128, seed=7)
        out, error = attend(pool, step, gpu_device)
        assert error == _hip.PAGED_ERANGE
        check(pool, step, out)
        pool.table = good


def test_pools_past_32_bits(gpu_device):
    # the sequence's pages lie behind 2^31 elements of the pool
    page, dim, kv = 64, 128, 2
    need = (1 << 31) // (kv * page * dim) + 40
    pool = Pool([90], kv, dim, page, seed=9, spare=0)
    small_k, small_v = pool.k.clone(), pool.v.clone()
    step = Step([10], [0], 8, dim, seed=9)
    q, starts, masks, rows = step.tensors(gpu_device)
    out = torch.full_like(q, 7.0)
    big = torch.zeros(2, need, kv, page, dim, dtype=torch.bfloat16, device=gpu_device)
    at = [need - 1 - i for i in range(small_k.shape[0])]
    big[0, at], big[1, at] = small_k.to(gpu_device), small_v.to(gpu_device)
    table = torch.tensor([at[int(p)] for p in pool.table[0]], dtype=I32)[None].to(gpu_device)
    error = flag(gpu_device)
    lengths = pool.lengths.to(gpu_device)
    _hip.paged_tree_attention(q, starts, masks, big[0], big[1], table, lengths, out,
                              workspace(step, pool, 64, 128, gpu_device), dim ** -0.5,
                              rows=rows, error_flag=error)
    check(pool, step, out.cpu())
    assert int(error.item()) == 0
    # and their rows move there
    ids, targets = torch.arange(10) + 100, torch.full((10,), 5)
    parents = [-1, 0, 0, 0, 3, 3, 3, 4, 5, 6]
    targets[0], targets[3], targets[5] = 103, 105, 108
    path = torch.zeros(1, 12, dtype=I32, device=gpu_device)
    counts, nxt = torch.zeros(1, dtype=I32, device=gpu_device), torch.zeros(
        1, dtype=I64, device=gpu_device)
    before = big[:, table[0].long()].clone()
    _hip.paged_tree_accept(starts, ids.to(gpu_device),
                           torch.tensor(parents, dtype=I32, device=gpu_device),
                           targets.to(gpu_device), path, counts, nxt, pages=big[None],
                           page_table=table, lengths=lengths, error_flag=error)
    assert path[0].tolist() == [0, 3, 5, 8] + [-1] * 8 and int(counts) == 4 and int(nxt) == 5
    after = big[:, table[0].long()]
    for j, node in enumerate((0, 3, 5, 8)):
        src, dst = 80 + node, 80 + j
        assert torch.equal(after[:, dst // page, :, dst % page],
                           before[:, src // page, :, src % page])
    assert int(error.item()) == 0


def test_another_stream_and_a_workspace_in_use_before(gpu_device):
    pool = Pool([1200, 400], 2, 128, 16, seed=11)
    step = Step([16, 9], [0, 1], 8, 128, seed=12)
    ws = workspace(step, pool, 64, pool.table.shape[1] * 16, gpu_device)
    first, _ = attend(pool, step, gpu_device, ws=ws)
    stream = torch.cuda.Stream(gpu_device)
    stream.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(stream):
        second, _ = attend(pool, step, gpu_device, ws=ws)
    assert torch.equal(first, second)
    check(pool, step, second)


def test_captured_attention_follows_the_device(gpu_device):
    # lengths, starts, masks and rows change between replays of one graph; the
    # eager call between them has a workspace of its own
    pool = Pool([700, 40, 9], 2, 128, 16, seed=13, width=50)
    step = Step([12, 5, 9], [0, 1, 2], 8, 128, seed=14)
    q, starts, masks, rows = step.tensors(gpu_device)
    k, v, table = (t.to(gpu_device) for t in (pool.k, pool.v, pool.table))
    lengths = pool.lengths.to(gpu_device)
    out, error = torch.full_like(q, 7.0), flag(gpu_device)
    ws = workspace(step, pool, 16, 800, gpu_device)

    def call(into, space):
        _hip.paged_tree_attention(q, starts, masks, k, v, table, lengths, into, space,
                                  128 ** -0.5, rows=rows, max_tree=16, error_flag=error)

    call(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws)
    other = torch.empty_like(ws)
    for lens, sizes, order in (([700, 40, 9], [12, 5, 9], [0, 1, 2]),
                               ([14, 33, 7], [3, 13, 7], [2, 0, -1]),
                               ([650, 25, 9], [1, 0, 14], [1, 2, 0])):
        fresh = Step(sizes, order, 8, 128, seed=sum(lens))
        pad = q.shape[0] - fresh.q.shape[0]
        fresh.masks += [0] * pad
        fresh.q = torch.cat((fresh.q, torch.zeros(pad, 8, 128, dtype=torch.bfloat16)))
        for old, new in zip((q, starts, masks, rows), fresh.tensors(gpu_device)):
            old.copy_(new)
        lengths.copy_(torch.tensor(lens, dtype=I32))
        pool.lengths = torch.tensor(lens, dtype=I32)
        out.fill_(7.0)
        graph.replay()
        replayed = out.clone()
        eager = torch.full_like(out, 7.0)
        call(eager, other)
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)
        fresh.masks = [m & (1 << 64) - 1 for m in fresh.masks]
        check(pool, fresh, replayed.cpu())
    assert int(error.item()) == 0


def test_two_calls_give_the_same_bits(gpu_device):
    pool = Pool([5000, 77, 2100], 2, 128, 64, seed=15)
    step = Step([20, 3, 64], [0, 1, 2], 8, 128, seed=16)
    first, _ = attend(pool, step, gpu_device)
    for _ in range(3):
        again, _ = attend(pool, step, gpu_device)
        assert torch.equal(first, again)


# ------------------------------------------------------------ acceptance


def accept_case(sizes, seed, vocab=4, chain=0.7):
    """ids, parents and targets of trees whose tokens repeat; some parents are
    none that can be followed."""

    rng = random.Random(seed)
    starts, ids, parents, targets = [0], [], [], []
    for n in sizes:
        mine = random_parents(n, rng, rng.choice((None, 2)))
        own = [rng.randrange(vocab) for _ in range(n)]
        drawn = []
        for i in range(n):
            children = [c for c in range(n) if mine[c] == i]
            if children and rng.random() < chain:
                drawn.append(own[rng.choice(children)])
            else:
                drawn.append(rng.choice((rng.randrange(vocab), -1, 1 << 40)))
        for i in range(1, n):
            if rng.random() < 0.1:
                mine[i] = rng.choice((-1, i, n + 3, 64, -7, i + 1))
        ids += own
        parents += mine
        targets += drawn
        starts.append(len(ids))
    return starts, ids, parents, targets


def run_accept(device, starts, ids, parents, targets, width, **pages):
    trees = len(starts) - 1
    path = torch.full((trees, width), 7, dtype=I32, device=device)
    counts = torch.full((trees,), 7, dtype=I32, device=device)
    next_ids = torch.full((trees,), 7, dtype=I64, device=device)
    error = flag(device)
    got = _hip.paged_tree_accept(
        torch.tensor(starts, dtype=I32, device=device),
        torch.tensor(ids, dtype=I64, device=device),
        torch.tensor(parents, dtype=I32, device=device),
        torch.tensor(targets, dtype=I64, device=device), path, counts, next_ids,
        error_flag=error, **pages)
    assert got is path
    return path.tolist(), counts.tolist(), next_ids.tolist(), int(error.item())


def expected(starts, ids, parents, targets, width, skip=()):
    paths, counts, nexts = [], [], []
    for b in range(len(starts) - 1):
        part = slice(starts[b], starts[b + 1])
        path, nxt = walk(ids[part], parents[part], targets[part])
        if b in skip:
            path, nxt = [], -1
        paths.append(path + [-1] * (width - len(path)))
        counts.append(len(path))
        nexts.append(nxt)
    return paths, counts, nexts


@pytest.mark.parametrize("seed", range(6))
def test_paths(gpu_device, seed):
    rng = random.Random(seed)
    sizes = [rng.choice((0, 1, 2, 5, 16, 33, 63, 64)) for _ in range(rng.choice((1, 7, 90)))]
    sizes[0] = max(1, sizes[0])
    case = accept_case(sizes, seed, chain=rng.choice((0.5, 0.95)))
    got = run_accept(gpu_device, *case, 64)
    assert got == (*expected(*case, 64), 0)
    narrow = max(sizes)
    assert run_accept(gpu_device, *case, narrow) == (*expected(*case, narrow), 0)


def test_the_longest_path(gpu_device):
    case = ([0, 64], list(range(64)), list(range(-1, 63)), list(range(1, 65)))
    assert run_accept(gpu_device, *case, 64) == ([list(range(64))], [64], [64], 0)


def test_the_first_of_equal_children(gpu_device):
    case = ([0, 5], [9, 4, 4, 6, 6], [-1, 0, 0, 2, 1], [4, 6, 6, 0, 3])
    assert run_accept(gpu_device, *case, 5) == ([[0, 1, 4, -1, -1]], [3], [3], 0)


def test_no_nodes_at_all_on_another_stream(gpu_device):
    stream, other = torch.cuda.Stream(gpu_device), torch.cuda.Stream(gpu_device)
    path = torch.full((2, 5), 7, dtype=I32, device=gpu_device)
    counts = torch.full((2,), 7, dtype=I32, device=gpu_device)
    next_ids = torch.full((2,), 7, dtype=I64, device=gpu_device)
    starts = torch.zeros(3, dtype=I32, device=gpu_device)
    none, parents = (torch.zeros(0, dtype=t, device=gpu_device) for t in (I64, I32))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(gpu_device)
    with torch.cuda.graph(graph, stream=stream):
        with torch.cuda.stream(other):  # not the one that the call names
            _hip.paged_tree_accept(starts, none, parents, none, path, counts, next_ids,
                                   stream=stream)
    torch.cuda.synchronize(gpu_device)
    assert bool((path == 7).all()), "ran on the current stream"
    graph.replay()
    torch.cuda.synchronize(gpu_device)
    assert bool((path == -1).all() and (counts == 0).all() and (next_ids == -1).all())


def test_trees_out_of_range(gpu_device):
    case = accept_case([4, 3, 6], 5)
    for change, skip in ((lambda s: s.__setitem__(3, 99), [2]),
                         (lambda s: s.__setitem__(0, -2), [0]),
                         (lambda s: s.__setitem__(1, 8), [0, 1])):
        starts = list(case[0])
        change(starts)
        path, counts, nxt, error = run_accept(gpu_device, starts, *case[1:], 6)
        assert error == _hip.PAGED_ERANGE
        for b in range(3):
            if b in skip and not (b == 0 and starts[1] == 8):
                assert path[b] == [-1] * 6 and counts[b] == 0 and nxt[b] == -1
    # more nodes than the path holds
    path, counts, nxt, error = run_accept(gpu_device, *case, 5)
    want = expected(*case, 5, skip=[2])
    assert (path, counts, nxt, error) == (*want, _hip.PAGED_ERANGE)
    # padding
    starts, ids, parents, targets = case
    rows = torch.tensor([0, -1, 2], dtype=I32, device=gpu_device)
    got = run_accept(gpu_device, *case, 6, rows=rows)
    assert got == (*expected(*case, 6, skip=[1]), 0)


def moved(pool_of, table, lengths, rows, starts, paths):
    """What the pool holds afterwards: every row read before any is written."""

    want = pool_of.clone()
    page = pool_of.shape[4]
    for b, row in enumerate(rows):
        n = starts[b + 1] - starts[b]
        past = lengths[row] - n
        for j, node in enumerate(paths[b]):
            if node < 0:
                break
            src, dst = past + node, past + j
            want[:, :, table[row][dst // page], :, dst % page] = (
                pool_of[:, :, table[row][src // page], :, src % page])
    return want


@pytest.mark.parametrize("layers,kv,dim,page_size,trees", [
    (1, 1, 16, 8, 1), (3, 2, 64, 8, 5), (2, 8, 128, 64, 9), (5, 3, 112, 16, 3),
    (1, 5, 1024, 16, 4), (32, 8, 128, 16, 1)])
def test_rows_move(gpu_device, layers, kv, dim, page_size, trees):
    rng = random.Random(layers * dim + trees)
    sizes = [rng.choice((1, 7, 16, 40, 64)) for _ in range(trees)]
    case = accept_case(sizes, dim, chain=0.95)
    lengths = [rng.choice((0, 1, 5, 30, 77)) for _ in range(trees + 2)]
    rows = rng.sample(range(trees + 2), trees)
    for b, row in enumerate(rows):
        lengths[row] += sizes[b]
    counts = [-(-n // page_size) for n in lengths]
    order = rng.sample(range(sum(counts) + 3), sum(counts))
    width = max(counts)
    table, at = [], 0
    for count in counts:
        table.append(order[at:at + count] + [-1] * (width - count))
        at += count
    pool = torch.randn(layers, 2, sum(counts) + 3, kv, page_size, dim).to(torch.bfloat16)
    on = pool.to(gpu_device)
    got = run_accept(gpu_device, *case, 64, pages=on,
                     page_table=torch.tensor(table, dtype=I32, device=gpu_device),
                     lengths=torch.tensor(lengths, dtype=I32, device=gpu_device),
                     rows=torch.tensor(rows, dtype=I32, device=gpu_device))
    assert got == (*expected(*case, 64), 0)
    assert torch.equal(on.cpu(), moved(pool, table, lengths, rows, case[0], got[0]))


def test_moves_out_of_range_are_left_out(gpu_device):
    # nodes 0 - 2 - 3 of 4, past 6, pages of 8: slots 6, 7 | 8, 9
    case = ([0, 4], [1, 2, 3, 4], [-1, 0, 0, 2], [3, 0, 4, 9])
    pool = torch.randn(1, 2, 4, 1, 8, 16).to(torch.bfloat16)
    table = [[2, 0, -1]]

    def run(table=table, length=10, rows=None):
        on = pool.to(gpu_device)
        got = run_accept(gpu_device, *case, 8, pages=on,
                         page_table=torch.tensor(table, dtype=I32, device=gpu_device),
                         lengths=torch.tensor([length], dtype=I32, device=gpu_device),
                         rows=None if rows is None else torch.tensor(
                             rows, dtype=I32, device=gpu_device))
        assert got[:3] == ([[0, 2, 3, -1, -1, -1, -1, -1]], [3], [9])
        return on.cpu(), got[3]

    on, error = run()
    want = pool.clone()
    want[:, :, 2, :, 7] = pool[:, :, 0, :, 0]
    want[:, :, 0, :, 0] = pool[:, :, 0, :, 1]
    assert error == 0 and torch.equal(on, want)
    for changes in (dict(length=3), dict(length=25), dict(length=-1), dict(rows=[1])):
        on, error = run(**changes)
        assert error == _hip.PAGED_ERANGE and torch.equal(on, pool)
    for bad in (-1, 4, 1 << 30):
        on, error = run(table=[[bad, 0, -1]])
        want = pool.clone()
        want[:, :, 0, :, 0] = pool[:, :, 0, :, 1]
        assert error == _hip.PAGED_ERANGE and torch.equal(on, want)


# ----------------------------------------------------------------- append


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_at_rope_rows_of_its_own(gpu_device, interleaved):
    g = torch.Generator().manual_seed(21)
    tokens, q_heads, kv, dim, page = 9, 4, 2, 64, 8
    q, k, v = (normal((tokens, h, dim), g) for h in (q_heads, kv, kv))
    cos, sin = normal((50, 16), g), normal((50, 16), g)
    positions = [3, 4, 5, 6, 7, 8, -1, 10, 11]
    turns = [3, 4, 4, 5, 49, 0, 2, 50, -1]  # the last two are outside the tables
    pools = torch.full((2, 6, kv, page, dim), 7.0, dtype=torch.bfloat16, device=gpu_device)
    table = torch.tensor([[4, 1]], dtype=I32, device=gpu_device)
    q_out = torch.full((tokens, q_heads, dim), 7.0, dtype=torch.bfloat16, device=gpu_device)
    error = flag(gpu_device)
    on = lambda x: torch.tensor(x, dtype=I32, device=gpu_device)
    _hip.paged_append(q.to(gpu_device), k.to(gpu_device), v.to(gpu_device), on(positions),
                      pools[0], pools[1], table, rows=on([0] * tokens),
                      rope=(cos.to(gpu_device), sin.to(gpu_device)),
                      interleaved=interleaved, q_out=q_out, error_flag=error,
                      rope_at=on(turns))
    assert int(error.item()) == _hip.PAGED_ERANGE
    pools, q_out = pools.cpu(), q_out.cpu()
    written = torch.zeros(6, page, dtype=torch.bool)
    for t, (pos, turn) in enumerate(zip(positions, turns)):
        if pos < 0 or not 0 <= turn < 50:
            assert bool((q_out[t] == 7).all())
            continue
        at = [4, 1][pos // page], pos % page
        written[at] = True
        for x, got in ((q[t], q_out[t]), (k[t], pools[0][at[0], :, at[1]])):
            ref, tol = rotated(x[None], cos[turn][None], sin[turn][None], interleaved)
            assert bool(((got.double() - ref[0]).abs() <= tol[0]).all())
        assert torch.equal(pools[1][at[0], :, at[1]], v[t])
    # [pages, slots, ..] views: everything else stays
    rest = pools.permute(1, 3, 0, 2, 4)[~written]
    assert bool((rest == 7).all())


# ------------------------------------------------------------------ steps


def test_drafted_steps_write_what_single_tokens_write(gpu_device):
    """Two sequences over several steps: a tree is appended, attended to and
    accepted, and the cache goes on with the accepted nodes.  Keys, values and
    the outputs of the accepted nodes are those of a second cache that got the
    accepted tokens one by one."""

    layers, q_heads, kv, dim, page, vocab = 2, 8, 2, 64, 8, 5
    g = torch.Generator().manual_seed(31)
    rng = random.Random(31)
    # a token's rows depend on its id and layer; its text position by rotation
    table_of = normal((layers, vocab, q_heads + 2 * kv, dim), g).to(gpu_device)
    angle = torch.arange(200, dtype=torch.float64)[:, None] * 0.3 ** torch.arange(32)
    rope = tuple(f.to(torch.bfloat16).to(gpu_device) for f in (angle.cos(), angle.sin()))
    caches = [PagedKVCache(40, 4, 200, layer_count=layers, num_kv_heads=kv, head_dim=dim,
                           page_size=page, device=gpu_device) for _ in range(2)]
    on = lambda x, dtype=I32: torch.tensor(x, dtype=dtype, device=gpu_device)

    def rows_of(layer, ids):
        return table_of[layer, on(ids, I64)]

    def single(cache, row, token):
        cache.extend([row])
        position = cache.length(row) - 1
        outs = []
        for layer in range(layers):
            x = rows_of(layer, [token])
            q = x[:, :q_heads].contiguous()
            cache.append(layer, q, x[:, q_heads:q_heads + kv], x[:, q_heads + kv:],
                         on([position]), rows=on([row]), rope=rope)
            out = torch.empty_like(q)
            cache.attend(layer, q, out, rows=on([row]))
            outs.append(out[0])
        return outs

    texts = [[0, 1, 2], [3]]
    rows = [[c.add() for _ in texts] for c in caches]
    rows[0] = [caches[0].fork(rows[0][0])[0], rows[0][1]]  # (row 0 stays empty)
    for s, text in enumerate(texts):
        for token in text:
            for c in range(2):
                single(caches[c], rows[c][s], token)
    # a sequence that shares the first one's pages, which drafts may not touch
    kept = caches[0].fork(rows[0][0])[0]
    snapshot = caches[0].buffer[:, :, caches[0].pages(kept)].clone()
    current = [4, 1]
    for step in range(6):
        sizes = [rng.choice((1, 6, 20)) for _ in texts]
        starts, ids, parents, targets, positions, turns, seq, masks = [0], [], [], [], [], [], [], []
        for s, n in enumerate(sizes):
            past = caches[0].length(rows[0][s])
            tree = random_parents(n, rng, 2)
            mask, depth = tree_masks(tree)
            own = [current[s]] + [rng.randrange(vocab) for _ in range(n - 1)]
            ids += own
            parents += tree
            masks += mask
            targets += [rng.randrange(vocab) for _ in range(n)]
            positions += range(past, past + n)
            turns += [past + d for d in depth]
            seq += [rows[0][s]] * n
            starts.append(len(ids))
            caches[0].extend([rows[0][s]], n)
        outs = []
        for layer in range(layers):
            x = rows_of(layer, ids)
            q = x[:, :q_heads].contiguous()
            caches[0].append(layer, q, x[:, q_heads:q_heads + kv], x[:, q_heads + kv:],
                             on(positions), rows=on(seq), rope=rope, rope_at=on(turns))
            out = torch.empty_like(q)
            caches[0].attend_tree(layer, q, on(starts), on(masks, I64), out,
                                  rows=on(rows[0]), max_tree=20)
            outs.append(out)
        path = torch.zeros(2, 20, dtype=I32, device=gpu_device)
        counts = torch.zeros(2, dtype=I32, device=gpu_device)
        next_ids = torch.zeros(2, dtype=I64, device=gpu_device)
        caches[0].accept(on(starts), on(ids, I64), on(parents), on(targets, I64), path,
                         counts, next_ids, rows=on(rows[0]))
        caches[0].check()
        for s, n in enumerate(sizes):
            count = int(counts[s])
            caches[0].truncate(rows[0][s], caches[0].length(rows[0][s]) - n + count)
            for j in range(count):
                node = starts[s] + int(path[s, j])
                for layer, out in enumerate(single(caches[1], rows[1][s], ids[node])):
                    off = (out.float() - outs[layer][node].float()).abs()
                    # one rounding of either output, and their weights'
                    assert bool((off <= 2.0 ** -7 * out.float().abs() + 2.0 ** -9).all())
            current[s] = int(next_ids[s])
    for s in range(2):
        length = caches[0].length(rows[0][s])
        assert length == caches[1].length(rows[1][s])
        flat = []
        for c in range(2):
            x = caches[c].buffer[:, :, caches[c].pages(rows[c][s])]
            flat.append(x.permute(0, 1, 3, 2, 4, 5).reshape(layers, 2, kv, -1, dim)[..., :length, :])
        assert torch.equal(*flat)
    assert torch.equal(caches[0].buffer[:, :, caches[0].pages(kept)][..., :3, :],
                       snapshot[..., :3, :])
