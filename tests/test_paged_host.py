"""The paged cache's bookkeeping, and every refusal of its operators and of
sampling, on the CPU: nothing here launches a kernel."""

import ctypes

import pytest
import torch

from layer_streaming import PagedKVCache, SimpleKVCache, _hip, paged

I32 = torch.int32


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose page copies are made by torch."""

    def copy(pages, pairs, error_flag=None, stream=None):
        src, dst = pairs[:, 0].tolist(), pairs[:, 1].tolist()
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        pages[:, :, dst] = pages[:, :, src]
        return pages

    monkeypatch.setattr(paged._hip, "copy_pages", copy)
    out = PagedKVCache(12, 5, 40, layer_count=2, num_kv_heads=1, head_dim=16, page_size=8,
                       device="cpu")
    # page p of plane j holds 100 j + p
    for layer in range(2):
        for which in (0, 1):
            for page in range(12):
                out.buffer[layer, which, page] = 100 * (2 * layer + which) + page
    return out


def consistent(cache):
    held = [p for pages in cache._pages if pages for p in pages]
    for page in range(cache.num_pages):
        assert cache._refs[page] == held.count(page)
    assert sorted(cache._free) == [p for p in range(cache.num_pages) if p not in held]
    for row in range(cache.max_sequences):
        pages = cache._pages[row] or []
        length = cache._lengths[row] if pages else 0
        assert cache.page_table[row].tolist() == pages + [-1] * (cache.max_pages - len(pages))
        assert int(cache.lengths[row]) == length
        assert len(pages) == -(-length // cache.page_size)


def test_extend_and_free(cache):
    a, b = cache.add(), cache.add()
    assert (a, b) == (0, 1)
    cache.extend([a], 9)
    cache.extend([b], 8)
    cache.extend([a, b])
    consistent(cache)
    assert cache.length(a) == 10 and cache.length(b) == 9
    assert cache.pages(a) == [0, 1] and cache.pages(b) == [2, 3]
    cache.free(a)
    consistent(cache)
    assert cache.free_pages == 10
    with pytest.raises(ValueError):
        cache.length(a)
    c = cache.add()
    assert c == a
    cache.extend([c], 1)
    assert cache.pages(c) == [0]
    consistent(cache)


def test_fork_copies_a_page_on_its_first_write(cache):
    a = cache.add()
    cache.extend([a], 13)
    b, c = cache.fork(a, 2)
    consistent(cache)
    assert cache.pages(a) == cache.pages(b) == [0, 1] and cache.free_pages == 10
    cache.extend([b])
    assert cache.pages(b) == [0, 2] and cache.pages(a) == [0, 1]
    assert float(cache.buffer[1, 0, 2, 0, 0, 0]) == 201  # page 1's content
    # the last two writers of a shared page: one copies, one keeps it
    cache.extend([a, c])
    assert cache.pages(a) == [0, 3] and cache.pages(c) == [0, 1]
    consistent(cache)
    # nothing is shared any more but the full page
    before = cache.free_pages
    cache.extend([a, b, c])
    assert cache.free_pages == before
    cache.truncate(b, 8)
    consistent(cache)
    assert cache.pages(b) == [0]
    # a write behind a full shared page takes a new page
    cache.extend([b])
    assert cache.pages(b) == [0, 2] and cache._refs[0] == 3
    # into a shared page after a truncation: copied
    cache.truncate(c, 5)
    cache.extend([c], 2)
    assert cache.pages(c) != [0] and cache.length(c) == 7
    consistent(cache)


def test_compact_moves_pages_to_the_front(cache):
    rows = [cache.add() for _ in range(4)]
    for row in rows:
        cache.extend([row], 20)
    forked = cache.fork(rows[3])[0]
    cache.free(rows[0])
    cache.free(rows[2])
    content = {r: [float(cache.buffer[1, 1, p, 0, 0, 0]) for p in cache.pages(r)]
               for r in (rows[1], rows[3], forked)}
    assert cache.compact() == 3
    consistent(cache)
    assert max(cache.pages(rows[1]) + cache.pages(rows[3])) == 5
    assert cache.pages(forked) == cache.pages(rows[3])
    for row, values in content.items():
        assert [float(cache.buffer[1, 1, p, 0, 0, 0]) for p in cache.pages(row)] == values
    assert cache.compact() == 0


def test_refusals_change_nothing(cache):
    a = cache.add()
    cache.extend([a], 39)
    for bad in (lambda: cache.extend([a], 2), lambda: cache.extend([a, a]),
                lambda: cache.extend([a, 3]), lambda: cache.extend([a], 0),
                lambda: cache.truncate(a, 40), lambda: cache.truncate(a, -1),
                lambda: cache.fork(a, 5), lambda: cache.free(2), lambda: cache.pages(-1),
                lambda: cache.pages(5)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
        consistent(cache)
        assert cache.length(a) == 39 and cache.free_pages == 7
    b = cache.add()
    cache.extend([b], 40)
    c = cache.add()
    with pytest.raises(RuntimeError):
        cache.extend([c], 24)  # 3 pages, 2 free
    consistent(cache)
    assert cache.length(c) == 0
    d, e = cache.add(), cache.add()
    with pytest.raises(RuntimeError):
        cache.add()
    for bad in (dict(page_size=12), dict(page_size=4), dict(page_size=2048),
                dict(num_pages=0), dict(max_length=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**dict(dict(num_pages=4, max_sequences=1, max_length=8,
                                     device="cpu"), **bad))


def test_rows_given_as_tensor_elements(cache):
    a, b = cache.add(), cache.add()
    cache.extend(torch.tensor([a, b]), 39)
    consistent(cache)
    with pytest.raises(ValueError):  # two tensors, one sequence
        cache.extend(torch.tensor([b, b]))
    consistent(cache)
    assert cache.length(b) == 39


def test_no_page_is_assigned_under_capture(cache, monkeypatch):
    a = cache.add()
    cache.extend([a], 20)
    b = cache.fork(a)[0]
    cache.free(a)
    monkeypatch.setattr(cache, "device", torch.device("cuda"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: cache.extend([b]), lambda: cache.fork(b), lambda: cache.free(b),
                 lambda: cache.truncate(b, 3), cache.compact):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    consistent(cache)
    assert cache.length(b) == 20


def test_load_refuses_another_geometry(cache):
    other = SimpleKVCache(2, 1, 32, device="cpu")
    other.append(0, torch.zeros(1, 1, 3, 32), torch.zeros(1, 1, 3, 32))
    with pytest.raises(ValueError):
        cache.load(cache.add(), other)
    # one layer behind the others
    other = SimpleKVCache(2, 1, 16, device="cpu")
    other.append(0, torch.zeros(1, 1, 3, 16), torch.zeros(1, 1, 3, 16))
    with pytest.raises(ValueError):
        cache.load(0, other)
    assert cache.length(0) == 0
    empty = SimpleKVCache(2, 1, 32, device="cpu")
    cache.load(0, empty)  # nothing to copy


def test_host_tensors_never_reach_a_kernel():
    z = torch.zeros
    bf = torch.bfloat16
    pool = z(3, 2, 8, 64, dtype=bf)
    k = z(1, 2, 64, dtype=bf)
    with pytest.raises(ValueError):
        _hip.paged_append(None, k, k, z(1, dtype=I32), pool, pool, z(1, 2, dtype=I32))
    with pytest.raises(ValueError):
        _hip.paged_decode_attention(z(1, 4, 64, dtype=bf), pool, pool, z(1, 2, dtype=I32),
                                    z(1, dtype=I32), z(1, 4, 64, dtype=bf),
                                    z(256, dtype=torch.uint8), 0.1)
    with pytest.raises(ValueError):
        _hip.copy_pages(z(2, 2, 3, 2, 8, 64), z(1, 2, dtype=I32))
    with pytest.raises(ValueError):
        _hip.sample(z(1, 10), z(1), z(1, dtype=torch.int64), z(256, dtype=torch.uint8))
    with pytest.raises(TypeError):
        _hip.sample(None, z(1), z(1, dtype=torch.int64), z(256, dtype=torch.uint8))


def append_args(**changes):
    names = dict(q=16, qt=1024, qh=128, k=16, kt=1024, kh=128, v=16, vt=1024, vh=128,
                 tokens=4, heads=8, kv=2, dim=128, positions=16, rows=16, table=16,
                 table_stride=10, sequences=4, max_pages=10, cos=16, sin=16,
                 rope_positions=100, rope_dim=128, interleaved=0, q_out=16, qot=1024,
                 qoh=128, k_pages=16, v_pages=16, page_stride=2 * 16 * 128,
                 head_stride=16 * 128, num_pages=20, page_size=16, error=16, stream=None)
    assert set(changes) <= set(names)
    names.update(changes)
    return list(names.values())


@pytest.mark.parametrize("code,changes", [
    (1001, dict(k=None)), (1001, dict(v_pages=None)), (1001, dict(positions=None)),
    (1001, dict(table=None)), (1001, dict(q=None)), (1001, dict(q_out=None)),
    (1001, dict(tokens=0)), (1001, dict(kv=0)), (1001, dict(heads=-1)),
    (1001, dict(table_stride=9)), (1001, dict(num_pages=0)), (1001, dict(cos=None)),
    (1001, dict(rope_positions=0)), (1001, dict(page_stride=16 * 128)),
    (1001, dict(head_stride=8 * 128)), (1003, dict(dim=120)), (1003, dict(page_size=24)),
    (1003, dict(page_size=4)), (1003, dict(page_size=2048, page_stride=1 << 20,
                                           head_stride=1 << 19)),
    (1003, dict(rope_dim=136)), (1003, dict(rope_dim=24)), (1003, dict(rope_dim=-16)),
    (1003, dict(max_pages=1 << 28, table_stride=1 << 28)),
    (1003, dict(max_pages=1 << 60, table_stride=1 << 60)),
    (1003, dict(tokens=1 << 25)), (1002, dict(k=24)),
    (1002, dict(q_out=8)), (1002, dict(cos=20)), (1002, dict(kt=1028)),
    (1002, dict(qh=-128)), (1002, dict(positions=18)), (1002, dict(error=17))])
def test_append_entry_point_refuses(code, changes):
    assert _hip.load().cascade_paged_append_bf16(*append_args(**changes)) == code


def attention_args(**changes):
    names = dict(q=16, qt=1024, qh=128, k_pages=16, v_pages=16, page_stride=2 * 16 * 128,
                 head_stride=16 * 128, num_pages=20, page_size=16, table=16,
                 table_stride=10, sequences=4, lengths=16, rows=16, batch=4, max_length=160,
                 heads=8, kv=2, dim=128, scale=ctypes.c_float(0.1), out=16, ot=1024, oh=128,
                 workspace=16, workspace_bytes=1 << 30, error=16, stream=None)
    assert set(changes) <= set(names)
    names.update(changes)
    return list(names.values())


@pytest.mark.parametrize("code,changes", [
    (1001, dict(q=None)), (1001, dict(lengths=None)), (1001, dict(workspace=None)),
    (1001, dict(batch=0)), (1001, dict(kv=0)), (1001, dict(max_length=0)),
    (1001, dict(max_length=161)), (1001, dict(page_stride=16 * 128)),
    (1001, dict(sequences=0)), (1003, dict(dim=96)), (1003, dict(heads=9)),
    (1003, dict(batch=1024, kv=8000, heads=128000, page_stride=8000 * 16 * 128,
                max_length=16000, table_stride=1000)),
    (1003, dict(heads=34)), (1003, dict(page_size=48)), (1003, dict(batch=1 << 24)), (1002, dict(q=20)),
    (1002, dict(out=8)), (1002, dict(qt=1020)), (1002, dict(lengths=18)),
    (1002, dict(workspace=8)), (1004, dict(workspace_bytes=8))])
def test_attention_entry_point_refuses(code, changes):
    fn = _hip.load().cascade_paged_decode_attention_bf16
    assert fn(*attention_args(**changes)) == code


def test_attention_workspace_shapes():
    assert _hip.paged_attention_workspace_bytes(1, 32, 8, 128, 1) > 0
    for bad in ((0, 32, 8, 128, 1), (1, 32, 8, 128, 0), (1, 33, 8, 128, 1),
                (1, 17, 1, 128, 1), (1, 32, 8, 80, 1)):
        with pytest.raises(ValueError):
            _hip.paged_attention_workspace_bytes(*bad)


@pytest.mark.parametrize("code,changes", [
    (1001, dict(pages=None)), (1001, dict(pairs=None)), (1001, dict(planes=0)),
    (1001, dict(num_pages=0)), (1001, dict(page_bytes=0)), (1001, dict(count=0)),
    (1001, dict(plane_bytes=9 * 4096)), (1002, dict(pages=8)), (1002, dict(page_bytes=4088)),
    (1002, dict(pairs=18)), (1002, dict(error=18))])
def test_copy_entry_point_refuses(code, changes):
    names = dict(pages=16, planes=2, plane_bytes=10 * 4096, num_pages=10, page_bytes=4096,
                 pairs=16, count=3, error=16, stream=None)
    names.update(changes)
    assert _hip.load().cascade_copy_pages(*names.values()) == code


@pytest.mark.parametrize("code,changes", [
    (1001, dict(logits=None)), (1001, dict(uniform=None)), (1001, dict(ids=None)),
    (1001, dict(workspace=None)), (1001, dict(rows=0)), (1001, dict(vocab=0)),
    (1001, dict(row_stride=99)), (1001, dict(t=-1.0)), (1001, dict(t=float("nan"))),
    (1001, dict(p=float("nan"))), (1001, dict(p=-0.5)), (1001, dict(m=-0.5)),
    (1003, dict(vocab=(1 << 19) + 1, row_stride=1 << 20)), (1003, dict(rows=1 << 23)), (1002, dict(ids=12)),
    (1002, dict(logits=18)), (1002, dict(workspace=8)), (1004, dict(workspace_bytes=8))])
def test_sample_entry_point_refuses(code, changes):
    names = dict(logits=16, row_stride=100, rows=2, vocab=100, uniform=16, t_ptr=None, t=1.0,
                 k_ptr=None, k=0, p_ptr=None, p=1.0, m_ptr=None, m=0.0, ids=16, logprobs=None,
                 workspace=16, workspace_bytes=1 << 30, stream=None)
    names.update(changes)
    assert _hip.load().cascade_sample_f32(*names.values()) == code


def test_workspaces_serve_smaller_calls_too():
    # sized once for the largest call: fewer rows never need more
    size = _hip.paged_attention_workspace_bytes
    for limit in (1, 500, 5000, 1 << 20):
        needs = [size(b, 32, 8, 128, limit) for b in (1, 2, 7, 64, 1000, 1024, 1025, 5000)]
        assert needs == sorted(needs)
    for vocab in (100, 16385, 20000, 128256, 1 << 19):
        needs = [_hip.sample_workspace_bytes(r, vocab) for r in range(1, 300)]
        assert needs == sorted(needs)


def test_sample_workspace_shapes():
    assert _hip.sample_workspace_bytes(1, 1) > 0
    assert _hip.sample_workspace_bytes(64, 1 << 19) > 0
    for rows, vocab in ((0, 10), (1, 0), (1, (1 << 19) + 1)):
        with pytest.raises(ValueError):
            _hip.sample_workspace_bytes(rows, vocab)
