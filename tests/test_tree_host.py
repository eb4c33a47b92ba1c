"""Drafted trees on the CPU: their masks, and what the operators refuse.  No
kernel is launched."""

import ctypes
import random

import pytest
import torch

from layer_streaming import PagedKVCache, _hip, tree_masks
from tree_cases import random_parents, signed

BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64


def test_masks_are_ancestors():
    rng = random.Random(1)
    for nodes in (0, 1, 2, 5, 33, 63, 64):
        parents = random_parents(nodes, rng)
        masks, depths = tree_masks(parents)
        assert len(masks) == len(depths) == nodes
        for node in range(nodes):
            line, at = 0, node
            depth = -1
            while at >= 0:
                line |= 1 << at
                at = parents[at]
                depth += 1
            assert masks[node] == signed(line) and depths[node] == depth
    masks, depths = tree_masks(range(-1, 63))
    assert masks[63] == -1 and depths[63] == 63
    torch.tensor(masks, dtype=I64)


@pytest.mark.parametrize("parents", [[0], [-1, -1], [-1, 1], [-1, 0, 3], [-1, -2],
                                     list(range(-1, 64))])
def test_no_tree(parents):
    with pytest.raises(ValueError):
        tree_masks(parents)


def test_parents_are_whole_numbers():
    with pytest.raises(TypeError):
        tree_masks([-1, 0.5])


def attention_args(**changes):
    names = dict(q=16, qt=1024, qh=128, tokens=9, starts=16, masks=16, trees=4, max_tree=8,
                 k_pages=16, v_pages=16, page_stride=2 * 16 * 128, head_stride=16 * 128,
                 num_pages=20, page_size=16, table=16, table_stride=10, sequences=4,
                 lengths=16, rows=16, max_length=160, heads=8, kv=2, dim=128,
                 scale=ctypes.c_float(0.1), out=16, ot=1024, oh=128, workspace=16,
                 workspace_bytes=1 << 30, error=16, stream=None)
    assert set(changes) <= set(names)
    names.update(changes)
    return list(names.values())


@pytest.mark.parametrize("code,changes", [
    (1001, dict(q=None)), (1001, dict(starts=None)), (1001, dict(masks=None)),
    (1001, dict(lengths=None)), (1001, dict(workspace=None)), (1001, dict(out=None)),
    (1001, dict(table=None)), (1001, dict(tokens=0)), (1001, dict(trees=0)),
    (1001, dict(tokens=1 << 31)), (1001, dict(max_tree=0)), (1001, dict(kv=0)),
    (1001, dict(max_length=0)), (1001, dict(max_length=161)),
    (1001, dict(page_stride=16 * 128)), (1001, dict(sequences=0)),
    (1001, dict(num_pages=0)), (1003, dict(max_tree=65)), (1003, dict(trees=1 << 20)),
    (1003, dict(dim=96)), (1003, dict(heads=9)), (1003, dict(heads=34)),
    (1003, dict(page_size=48)), (1003, dict(max_length=1 << 31, table_stride=1 << 31)),
    (1002, dict(q=20)), (1002, dict(out=8)), (1002, dict(qt=1020)), (1002, dict(oh=-128)),
    (1002, dict(starts=18)), (1002, dict(masks=20)), (1002, dict(lengths=18)),
    (1002, dict(rows=17)), (1002, dict(workspace=8)), (1002, dict(error=18)),
    (1004, dict(workspace_bytes=8))])
def test_attention_entry_point_refuses(code, changes):
    fn = _hip.load().cascade_paged_tree_attention_bf16
    assert fn(*attention_args(**changes)) == code


def test_attention_workspace_shapes():
    size = _hip.paged_tree_attention_workspace_bytes
    assert size(1, 1, 32, 8, 128, 1) > 0
    for bad in ((0, 8, 32, 8, 128, 1), (1, 0, 32, 8, 128, 1), (1, 65, 32, 8, 128, 1),
                (1, 8, 32, 8, 128, 0), (1, 8, 33, 8, 128, 1), (1, 8, 17, 1, 128, 1),
                (1, 8, 32, 8, 80, 1)):
        with pytest.raises(ValueError):
            size(*bad)
    # sized once for the largest call: smaller ones never need more
    for limit in (1, 500, 5000, 1 << 20):
        for nodes in (1, 4, 16, 64):
            needs = [size(b, nodes, 32, 8, 128, limit) for b in (1, 2, 7, 64, 300, 1025)]
            assert needs == sorted(needs)
        needs = [size(3, nodes, 32, 8, 128, limit) for nodes in range(1, 65)]
        assert needs == sorted(needs)
    needs = [size(3, 16, 32, 8, 128, n) for n in range(1, 3000, 7)]
    assert needs == sorted(needs)


def accept_args(**changes):
    names = dict(starts=16, ids=16, parents=16, targets=16, tokens=9, trees=3, max_tree=8,
                 path=16, counts=16, next_ids=16, pages=16, planes=4,
                 plane_bytes=20 * 2 * 16 * 256, num_pages=20, kv=2, page_size=16,
                 row_bytes=256, table=16, table_stride=10, sequences=4, max_pages=10,
                 lengths=16, rows=16, error=16, stream=None)
    assert set(changes) <= set(names)
    names.update(changes)
    return list(names.values())


@pytest.mark.parametrize("code,changes", [
    (1001, dict(starts=None)), (1001, dict(ids=None)), (1001, dict(parents=None)),
    (1001, dict(targets=None)), (1001, dict(path=None)), (1001, dict(counts=None)),
    (1001, dict(next_ids=None)), (1001, dict(tokens=0)), (1001, dict(trees=0)),
    (1001, dict(max_tree=0)), (1001, dict(table=None)), (1001, dict(lengths=None)),
    (1001, dict(planes=0)), (1001, dict(num_pages=0)), (1001, dict(kv=0)),
    (1001, dict(row_bytes=0)), (1001, dict(sequences=0)), (1001, dict(table_stride=9)),
    (1001, dict(plane_bytes=19 * 2 * 16 * 256)), (1003, dict(max_tree=65)),
    (1003, dict(page_size=24)), (1003, dict(kv=1025)), (1003, dict(row_bytes=4096)),
    (1003, dict(trees=1 << 25)), (1003, dict(planes=1 << 20)),
    (1003, dict(max_pages=1 << 60, table_stride=1 << 60)),
    (1002, dict(starts=18)), (1002, dict(ids=20)), (1002, dict(parents=17)),
    (1002, dict(targets=20)), (1002, dict(path=18)), (1002, dict(counts=18)),
    (1002, dict(next_ids=20)), (1002, dict(pages=8)), (1002, dict(row_bytes=264)),
    (1002, dict(table=18)), (1002, dict(rows=18)), (1002, dict(error=18))])
def test_accept_entry_point_refuses(code, changes):
    assert _hip.load().cascade_paged_tree_accept(*accept_args(**changes)) == code


def test_turned_append_refuses_an_unaligned_row_vector():
    args = [16, 1024, 128, 16, 1024, 128, 16, 1024, 128, 4, 8, 2, 128, 16, 18, 16, 16, 10, 4,
            10, 16, 16, 100, 128, 0, 16, 1024, 128, 16, 16, 2 * 16 * 128, 16 * 128, 20, 16,
            16, None]
    assert _hip.load().cascade_paged_append_turned_bf16(*args) == 1002


# ---------------------------------------------------------------- wrappers


def attention_call(device):
    z = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.paged_tree_attention, dict(
        q=z(5, 4, 64), starts=z(4, dtype=I32), masks=z(5, dtype=I64),
        k_pages=z(5, 2, 8, 64), v_pages=z(5, 2, 8, 64), page_table=z(4, 3, dtype=I32),
        lengths=z(4, dtype=I32), out=z(5, 4, 64), workspace=z(4096, dtype=torch.uint8),
        scale=0.125, rows=z(3, dtype=I32), max_tree=8, max_length=24,
        error_flag=z(1, dtype=I32))


def accept_call(device):
    z = lambda *shape, dtype=I32: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.paged_tree_accept, dict(
        starts=z(4), ids=z(5, dtype=I64), parents=z(5), targets=z(5, dtype=I64),
        path=z(3, 8), counts=z(3), next_ids=z(3, dtype=I64),
        pages=z(2, 2, 5, 2, 8, 64, dtype=BF), page_table=z(4, 3), lengths=z(4), rows=z(3),
        error_flag=z(1))


def append_call(device):
    z = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.paged_append, dict(
        q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), positions=z(3, dtype=I32),
        k_pages=z(5, 2, 8, 64), v_pages=z(5, 2, 8, 64), page_table=z(4, 3, dtype=I32),
        rows=z(3, dtype=I32), rope=(z(24, 32), z(24, 32)), rope_at=z(3, dtype=I32))


CALLS = {"attention": attention_call, "accept": accept_call, "append": append_call}

_short = lambda t: t[:-1].contiguous()
_wide = lambda t: torch.stack((t, t), -1).flatten(-2)[..., ::2]

WRONG = [
    ("attention", "q", lambda t: t.float()), ("attention", "q", _short),
    ("attention", "q", _wide), ("attention", "q", lambda t: None),
    ("attention", "q", lambda t: t[..., :32].contiguous()),
    ("attention", "starts", lambda t: t.long()), ("attention", "starts", _wide),
    ("attention", "starts", lambda t: t[None]), ("attention", "starts", lambda t: t[:0]),
    ("attention", "starts", lambda t: torch.cat((t, t))), ("attention", "starts", lambda t: None),
    ("attention", "masks", lambda t: t.int()), ("attention", "masks", _short),
    ("attention", "masks", _wide), ("attention", "masks", lambda t: None),
    ("attention", "k_pages", lambda t: t.float()), ("attention", "v_pages", _short),
    ("attention", "k_pages", _wide), ("attention", "page_table", lambda t: t.long()),
    ("attention", "page_table", _wide), ("attention", "lengths", lambda t: t.long()),
    ("attention", "lengths", _short), ("attention", "out", lambda t: t.float()),
    ("attention", "out", _short), ("attention", "out", lambda t: t[:1].expand_as(t)),
    ("attention", "rows", _short), ("attention", "rows", lambda t: t.long()),
    ("attention", "workspace", lambda t: t.view(torch.int8)),
    ("attention", "workspace", _wide), ("attention", "max_tree", lambda t: 0),
    ("attention", "max_tree", lambda t: 65), ("attention", "max_tree", lambda t: 2.5),
    ("attention", "max_length", lambda t: 0), ("attention", "max_length", lambda t: 25),
    ("attention", "error_flag", lambda t: t.long()),
    ("accept", "starts", lambda t: t.long()), ("accept", "starts", lambda t: t[:0]),
    ("accept", "starts", _wide), ("accept", "ids", lambda t: t.int()), ("accept", "ids", _short),
    ("accept", "ids", _wide), ("accept", "parents", lambda t: t.long()),
    ("accept", "parents", _short), ("accept", "targets", lambda t: t.int()),
    ("accept", "targets", _short), ("accept", "path", lambda t: t.long()),
    ("accept", "path", _short), ("accept", "path", lambda t: t.t().contiguous().t()),
    ("accept", "path", lambda t: torch.zeros(3, 65, dtype=I32)),
    ("accept", "path", lambda t: t[:, :0]), ("accept", "counts", _short),
    ("accept", "counts", lambda t: t.long()), ("accept", "next_ids", lambda t: t.int()),
    ("accept", "next_ids", _short), ("accept", "pages", lambda t: t.float()),
    ("accept", "pages", lambda t: t[0]), ("accept", "pages", _wide),
    ("accept", "pages", lambda t: t[:, :1].contiguous()),
    ("accept", "page_table", lambda t: t.long()), ("accept", "page_table", lambda t: None),
    ("accept", "lengths", _short), ("accept", "lengths", lambda t: None),
    ("accept", "rows", _short), ("accept", "rows", lambda t: t.long()),
    ("accept", "pages", lambda t: None), ("accept", "error_flag", lambda t: t.long()),
    ("append", "rope_at", lambda t: t.long()), ("append", "rope_at", _short),
    ("append", "rope_at", _wide), ("append", "rope_at", lambda t: t[:, None]),
]


@pytest.fixture
def launches(monkeypatch):
    calls = []

    def on(name, tensor):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(name)
        return tensor.device

    monkeypatch.setattr(_hip, "_gpu_of", on)
    monkeypatch.setattr(_hip, "_call_on", lambda *args: calls.append(args))
    return calls


@pytest.mark.parametrize("which", CALLS)
def test_the_call_itself_is_taken(launches, which):
    function, args = CALLS[which]("cpu")
    function(**args)
    assert len(launches) == 1


@pytest.mark.parametrize("which,name,change", WRONG,
                         ids=["{}-{}-{}".format(i, *c[:2]) for i, c in enumerate(WRONG)])
def test_wrong_arguments_are_refused(launches, which, name, change):
    function, args = CALLS[which]("cpu")
    args[name] = change(args[name])
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert not launches


def test_more_trees_than_rows_need_row_numbers(launches):
    for which in ("attention", "accept"):
        function, args = CALLS[which]("cpu")
        args.update(rows=None, page_table=args["page_table"][:2].contiguous(),
                    lengths=args["lengths"][:2].contiguous())
        with pytest.raises(ValueError):
            function(**args)
    assert not launches


def test_no_trees_and_no_rows(launches):
    function, args = attention_call("cpu")
    for starts in (args["starts"][:1], args["starts"]):
        few = dict(args, starts=starts, rows=None)
        if starts.shape[0] > 1:
            few.update(q=args["q"][:0], masks=args["masks"][:0], out=args["out"][:0])
        assert function(**few) is few["out"]
    function, args = accept_call("cpu")
    for name in ("ids", "parents", "targets"):
        args[name] = args[name][:0]
    assert function(**args) is args["path"]
    assert args["path"].tolist() == [[-1] * 8] * 3 and args["counts"].tolist() == [0] * 3
    assert args["next_ids"].tolist() == [-1] * 3
    assert not launches


def test_acceptance_alone_needs_no_pages(launches):
    function, args = accept_call("cpu")
    args.update(pages=None, page_table=None, lengths=None)
    function(**args)
    assert len(launches) == 1


def test_the_caches_workspace_serves_trees_and_single_tokens():
    cache = PagedKVCache(num_pages=4, max_sequences=3, max_length=20, layer_count=1,
                         num_kv_heads=2, head_dim=64, page_size=8, device="cpu")
    need = _hip.paged_tree_attention_workspace_bytes(3, 64, 8, 2, 64, 24)
    held = cache._workspace(need)
    assert held.numel() >= need and cache._workspace(16) is held
    assert cache._attention_workspace(1, 8).numel() >= (
        _hip.paged_attention_workspace_bytes(1, 8, 2, 64, 24))


def test_heads_that_attention_does_not_take():
    cache = PagedKVCache(num_pages=4, max_sequences=3, max_length=20, layer_count=1,
                         num_kv_heads=2, head_dim=80, page_size=8, device="cpu")
    with pytest.raises(ValueError):
        cache.attend_tree(0, None, None, None, None)
