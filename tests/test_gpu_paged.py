"""The paged KV cache's operators against their plain 64-bit forms: rotary
positions with the write into pages, attention of one token a sequence, page
copies; and a decode step of several sequences made of them."""

import math

import pytest
import torch

from layer_streaming import PagedKVCache, SimpleKVCache, _hip
from paged_cases import Pool, attention, normal, rotated

pytestmark = pytest.mark.gpu


def workspace(batch, q_heads, kv_heads, dim, limit, device):
    size = _hip.paged_attention_workspace_bytes(batch, q_heads, kv_heads, dim, limit)
    return torch.full((size,), 0xFF, dtype=torch.uint8, device=device)


def flag(device):
    return torch.zeros(1, dtype=torch.int32, device=device)


def attend(pool, q, rows, device, limit=None, out=None, ws=None, error=None,
           q_view=None):
    """Run the operator over CPU inputs; returns (out on the CPU, flag)."""

    kv, dim = pool.k.shape[1], pool.k.shape[3]
    limit = pool.table.shape[1] * pool.k.shape[2] if limit is None else limit
    qd = q.to(device) if q_view is None else q_view
    out = torch.full_like(q, 7.0).to(device) if out is None else out
    error = flag(device) if error is None else error
    if ws is None:
        ws = workspace(q.shape[0], q.shape[1], kv, dim, limit, device)
    rows_d = None if rows is None else torch.tensor(rows, dtype=torch.int32, device=device)
    got = _hip.paged_decode_attention(
        qd, pool.k.to(device), pool.v.to(device), pool.table.to(device),
        pool.lengths.to(device), out, ws, dim ** -0.5, rows=rows_d, max_length=limit,
        error_flag=error)
    assert got is out
    torch.cuda.synchronize(device)
    return out.cpu(), int(error.item())


def check_attention(pool, q, rows, out, lengths=None):
    dim = q.shape[2]
    lengths = pool.lengths.tolist() if lengths is None else lengths
    rows = range(q.shape[0]) if rows is None else rows
    for b, row in enumerate(rows):
        if not 0 <= row < pool.table.shape[0]:
            assert bool((out[b] == 7.0).all()), "padding row {} was written".format(b)
            continue
        k, v, good = pool.rows_of(row, lengths[row])
        ref, tol = attention(q[b], k, v, good, dim ** -0.5)
        off = (out[b].double() - ref).abs()
        assert bool((off <= tol).all()), (b, row, lengths[row], float((off - tol).max()))


SHAPES = [(32, 8, 128), (5, 5, 64), (16, 1, 128), (12, 4, 64), (6, 2, 128), (48, 3, 64),
          (9, 1, 64)]


@pytest.mark.parametrize("q_heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("page_size", [8, 16, 64, 256])
def test_attention_lengths(gpu_device, q_heads, kv_heads, dim, page_size):
    print("attention", q_heads, kv_heads, dim, page_size, flush=True)
    lengths = [1, 0, 7, 8, 9, 31, 32, 33, 127, 128, 129, 257, 600, 1025]
    pool = Pool(lengths, kv_heads, dim, page_size, seed=page_size + q_heads)
    q = normal((len(lengths), q_heads, dim), torch.Generator().manual_seed(3), 2.0)
    out, error = attend(pool, q, None, gpu_device)
    check_attention(pool, q, None, out)
    assert bool((out[1] == 0).all()) and error == 0


@pytest.mark.parametrize("batch,length,page_size", [(1, 1, 8), (1, 40, 16), (1, 9000, 64),
                                                    (2, 5000, 16), (150, 70, 8),
                                                    (3, 20001, 128)])
def test_attention_batches(gpu_device, batch, length, page_size):
    print("attention batch", batch, length, page_size, flush=True)
    lengths = [max(0, length - 37 * i) for i in range(batch)]
    pool = Pool(lengths, 2, 128, page_size, seed=batch)
    q = normal((batch, 8, 128), torch.Generator().manual_seed(4), 1.5)
    out, error = attend(pool, q, None, gpu_device)
    check_attention(pool, q, None, out)
    assert error == 0


def test_attention_rows_padding_and_strides(gpu_device):
    # batch rows in another order, one sequence twice, padding rows, q and out
    # as views of wider rows, pools as views of a larger buffer
    lengths = [300, 5, 64, 0, 1000]
    pool = Pool(lengths, 4, 64, 16, seed=1, width=80)
    rows = [4, -1, 0, 2, 4, 3, -5, 1]
    g = torch.Generator().manual_seed(5)
    fused = normal((len(rows), 24, 64), g).to(gpu_device)
    q = fused[:, 3:15]
    wide = torch.full((len(rows), 20, 64), 7.0, dtype=torch.bfloat16, device=gpu_device)
    buffer = torch.stack((pool.k, pool.v)).to(gpu_device)  # [2, pages, ...]
    both = torch.stack((buffer, buffer)).transpose(1, 2).contiguous()
    ws = workspace(len(rows), 12, 4, 64, 1280, gpu_device)
    error = flag(gpu_device)
    out = wide[:, 4:16]
    _hip.paged_decode_attention(
        q, both[1, :, 0], both[1, :, 1], pool.table.to(gpu_device),
        pool.lengths.to(gpu_device), out, ws, 64 ** -0.5,
        rows=torch.tensor(rows, dtype=torch.int32, device=gpu_device), error_flag=error)
    check_attention(pool, q.cpu(), rows, out.cpu())
    assert bool((wide[:, :4] == 7).all()) and bool((wide[:, 16:] == 7).all())
    assert int(error.item()) == 0


def test_attention_flags_what_is_out_of_range(gpu_device):
    lengths = [100, 90, 80, 70]
    pool = Pool(lengths, 2, 128, 16, seed=2)
    q = normal((4, 8, 128), torch.Generator().manual_seed(6))
    # sequences past the table: left alone
    out, error = attend(pool, q, [0, 4, 1, 1 << 30], gpu_device)
    assert error == _hip.PAGED_ERANGE
    check_attention(pool, q, [0, 4, 1, 1 << 30], out)
    # pages outside the pool: their positions are left out
    pool.table[0, 2] = 10 ** 9
    pool.table[1, 5] = -1
    pool.table[2, :] = pool.k.shape[0]
    out, error = attend(pool, q, None, gpu_device)
    assert error == _hip.PAGED_ERANGE
    check_attention(pool, q, None, out)
    assert bool((out[2] == 0).all())
    # a length past max_length is cut to it, a negative one is empty
    pool = Pool(lengths, 2, 128, 16, seed=2)
    pool.lengths = torch.tensor([100, -3, 2 ** 31 - 1, 70], dtype=torch.int32)
    out, error = attend(pool, q, None, gpu_device, limit=75)
    assert error == _hip.PAGED_ERANGE
    check_attention(pool, q, None, out, lengths=[75, 0, 75, 70])


def test_attention_infinite_scores_and_nan(gpu_device):
    # an infinite or NaN value in the cache reaches the heads and sequences
    # that read it and no others
    lengths = [40, 40]
    pool = Pool(lengths, 2, 128, 16, seed=7)
    page = int(pool.table[0, 1])
    pool.k[page, 0, 3, 5] = math.nan
    pool.v[page, 1, 2, 9] = math.inf
    q = normal((2, 4, 128), torch.Generator().manual_seed(8))
    out, error = attend(pool, q, None, gpu_device)
    assert error == 0
    assert bool(out[0, :2].isnan().all())
    assert bool((out[0, 2:, 9] == math.inf).all())
    assert bool(out[0, 2:, :9].isfinite().all()) and bool(out[0, 2:, 10:].isfinite().all())
    k, v, good = pool.rows_of(1, 40)
    ref, tol = attention(q[1], k, v, good, 128 ** -0.5)
    assert bool(((out[1].double() - ref).abs() <= tol).all())


def test_attention_large_scores(gpu_device):
    # scores in the hundreds: one position takes all the weight
    pool = Pool([777], 1, 64, 32, seed=9)
    pool.k *= 12
    q = normal((1, 16, 64), torch.Generator().manual_seed(10), 12.0)
    out, _ = attend(pool, q, None, gpu_device)
    check_attention(pool, q, None, out)


def test_attention_repeats_bit_for_bit(gpu_device):
    pool = Pool([4000, 1, 900], 2, 128, 16, seed=11)
    q = normal((3, 8, 128), torch.Generator().manual_seed(12))
    first, _ = attend(pool, q, None, gpu_device)
    for _ in range(3):
        again, _ = attend(pool, q, None, gpu_device)
        assert torch.equal(first, again)


def test_attention_far_pages(gpu_device):
    # page offsets past 32 bits: a pool of 4.3e9 bytes, K and V interleaved
    pages, kv, page_size, dim = 16500, 8, 64, 128
    both = torch.zeros((pages, 2, kv, page_size, dim), dtype=torch.bfloat16,
                       device=gpu_device)
    pool = Pool([130], kv, dim, page_size, seed=13)
    far = [pages - 1, 3, pages - 2]
    for i, page in enumerate(far):
        both[page, 0] = pool.k[int(pool.table[0, i])].to(gpu_device)
        both[page, 1] = pool.v[int(pool.table[0, i])].to(gpu_device)
    q = normal((1, 32, dim), torch.Generator().manual_seed(14))
    out = torch.empty_like(q).to(gpu_device)
    table = torch.tensor([far], dtype=torch.int32, device=gpu_device)
    ws = workspace(1, 32, kv, dim, 192, gpu_device)
    _hip.paged_decode_attention(q.to(gpu_device), both[:, 0], both[:, 1], table,
                                pool.lengths.to(gpu_device), out, ws, dim ** -0.5)
    check_attention(pool, q, None, out.cpu())
    # the append to a far page
    k, v = normal((1, kv, dim), torch.Generator().manual_seed(15)), normal(
        (1, kv, dim), torch.Generator().manual_seed(16))
    _hip.paged_append(None, k.to(gpu_device), v.to(gpu_device),
                      torch.tensor([131], dtype=torch.int32, device=gpu_device),
                      both[:, 0], both[:, 1], table)
    assert torch.equal(both[far[2], 0, :, 3].cpu(), k[0])
    assert torch.equal(both[far[2], 1, :, 3].cpu(), v[0])


# ------------------------------------------------------------------- append


def append_case(tokens, heads, kv_heads, dim, rope_dim, page_size, seed, sequences=4):
    g = torch.Generator().manual_seed(seed)
    fused = normal((tokens, heads + 2 * kv_heads, dim), g, 3.0)
    limit = 4 * page_size + 40
    pool = Pool([limit] * sequences, kv_heads, dim, page_size, seed=seed)
    # distinct positions in random order over random sequences
    spots = torch.randperm(sequences * limit, generator=g)[:tokens]
    rows, positions = (spots // limit).tolist(), (spots % limit).tolist()
    cos = sin = None
    if rope_dim:
        angle = torch.rand((limit, rope_dim // 2), generator=g) * 6.3
        cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    return fused, pool, rows, positions, cos, sin


def check_append(fused, heads, kv_heads, pool, before, rows, positions, cos, sin,
                 interleaved, q_out, live):
    page_size = pool.k.shape[2]
    at = torch.tensor(positions).clamp(min=0)
    c, s = (None, None) if cos is None else (cos[at], sin[at])
    q_ref, q_tol = rotated(fused[:, :heads], c, s, interleaved)
    k_ref, k_tol = rotated(fused[:, heads:heads + kv_heads], c, s, interleaved)
    k_now, v_now = pool.k.clone(), pool.v.clone()
    for t in range(len(rows)):
        if t not in live:
            assert bool((q_out[t] == 7).all())
            continue
        assert bool(((q_out[t].double() - q_ref[t]).abs() <= q_tol[t]).all())
        page = int(pool.table[rows[t], positions[t] // page_size])
        slot = positions[t] % page_size
        assert bool(((k_now[page, :, slot].double() - k_ref[t]).abs() <= k_tol[t]).all())
        assert torch.equal(v_now[page, :, slot], fused[t, heads + kv_heads:])
        k_now[page, :, slot] = before.k[page, :, slot]
        v_now[page, :, slot] = before.v[page, :, slot]
    # nothing else was written (NaN where no sequence has a row)
    assert torch.equal(k_now.view(torch.int16), before.k.view(torch.int16))
    assert torch.equal(v_now.view(torch.int16), before.v.view(torch.int16))


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rope_dim,page_size", [
    (1, 32, 8, 128, 128, 16), (3, 32, 8, 128, 64, 64), (64, 5, 5, 64, 64, 8),
    (77, 7, 1, 128, 16, 32), (200, 12, 4, 64, 32, 16), (33, 4, 2, 96, 96, 16),
    (9, 3, 3, 16, 16, 8), (40, 2, 1, 256, 0, 128), (300, 32, 8, 128, 128, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(gpu_device, tokens, heads, kv_heads, dim, rope_dim, page_size, interleaved):
    print("append", tokens, heads, kv_heads, dim, rope_dim, page_size, flush=True)
    fused, pool, rows, positions, cos, sin = append_case(
        tokens, heads, kv_heads, dim, rope_dim, page_size, seed=tokens)
    padding = {1, 5, tokens - 1} if tokens > 8 else set()
    for t in padding:
        if t % 2:
            positions[t] = -1
        else:
            rows[t] = -1
    before = Pool([1], kv_heads, dim, page_size, seed=0)
    before.k, before.v = pool.k.clone(), pool.v.clone()
    dev = gpu_device
    pool.to(dev)
    f = fused.to(dev)
    q_out = torch.full((tokens, heads, dim), 7.0, dtype=torch.bfloat16, device=dev)
    error = flag(dev)
    got = _hip.paged_append(
        f[:, :heads], f[:, heads:heads + kv_heads], f[:, heads + kv_heads:],
        torch.tensor(positions, dtype=torch.int32, device=dev), pool.k, pool.v, pool.table,
        rows=torch.tensor(rows, dtype=torch.int32, device=dev),
        rope=None if cos is None else (cos.to(dev), sin.to(dev)),
        interleaved=interleaved, q_out=q_out, error_flag=error)
    assert got is q_out and int(error.item()) == 0
    pool.to("cpu")
    live = set(range(tokens)) - padding
    check_append(fused, heads, kv_heads, pool, before, rows, positions, cos, sin,
                 interleaved, q_out.cpu(), live)
    # in place: q_out left out
    again = _hip.paged_append(
        f[:, :heads], f[:, heads:heads + kv_heads], f[:, heads + kv_heads:],
        torch.tensor(positions, dtype=torch.int32, device=dev), pool.k.to(dev),
        pool.v.to(dev), pool.table.to(dev),
        rows=torch.tensor(rows, dtype=torch.int32, device=dev),
        rope=None if cos is None else (cos.to(dev), sin.to(dev)), interleaved=interleaved)
    for t in live:
        assert torch.equal(again[t], q_out[t])
    for t in padding:
        assert torch.equal(again[t].cpu(), fused[t, :heads])


def test_append_leaves_out_of_range_tokens_out(gpu_device):
    heads, kv, dim, page_size = 4, 2, 64, 16
    fused, pool, rows, positions, cos, sin = append_case(8, heads, kv, dim, 64, page_size, 3)
    dev = gpu_device
    before = Pool([1], kv, dim, page_size, seed=0)
    before.k, before.v = pool.k.clone(), pool.v.clone()
    capacity = pool.table.shape[1] * page_size
    rows[0] = 4                      # no such sequence
    positions[1] = capacity          # behind the table row
    positions[2] = 2 ** 31 - 1
    pool.table[3, :] = -1            # sequence 3 has no pages
    rows[3], positions[3] = 3, 5
    pool.table[2, 1] = pool.k.shape[0]
    rows[4], positions[4] = 2, 17
    cos, sin = cos[:-30], sin[:-30]  # positions 74.. have no rope row
    rows[5], positions[5] = 0, cos.shape[0]
    rows[6], positions[6] = 0, 3
    rows[7], positions[7] = 1, 0
    pool.to(dev)
    f = fused.to(dev)
    q_out = torch.full((8, heads, dim), 7.0, dtype=torch.bfloat16, device=dev)
    error = flag(dev)
    _hip.paged_append(f[:, :heads], f[:, heads:heads + kv], f[:, heads + kv:],
                      torch.tensor(positions, dtype=torch.int32, device=dev), pool.k, pool.v,
                      pool.table, rows=torch.tensor(rows, dtype=torch.int32, device=dev),
                      rope=(cos.to(dev), sin.to(dev)), q_out=q_out, error_flag=error)
    assert int(error.item()) == _hip.PAGED_ERANGE
    pool.to("cpu")
    clipped = [min(p, cos.shape[0] - 1) for p in positions]
    check_append(fused, heads, kv, pool, before, rows, clipped, cos, sin, False,
                 q_out.cpu(), {6, 7})


# ------------------------------------------------------------------- copies


@pytest.mark.parametrize("layers,pages,kv,page_size,dim", [
    (1, 9, 1, 8, 16), (3, 40, 8, 16, 128), (2, 12, 5, 64, 64), (32, 8, 8, 16, 128)])
def test_copy_pages(gpu_device, layers, pages, kv, page_size, dim):
    print("copy", layers, pages, kv, page_size, dim, flush=True)
    g = torch.Generator().manual_seed(pages)
    buffer = normal((layers, 2, pages, kv, page_size, dim), g)
    order = torch.randperm(pages, generator=g).tolist()
    pairs = [[order[2 * i], order[2 * i + 1]] for i in range(pages // 2)]
    # padding pairs, pages outside the pool, a page onto itself
    extra = [[-1, 0], [0, -7], [pages, 0], [0, pages], [2 ** 31 - 1, 1]]
    if pages % 2:
        extra.append([order[-1], order[-1]])
    expected = buffer.clone()
    for src, dst in pairs:
        expected[:, :, dst] = buffer[:, :, src]
    dev = gpu_device
    error = flag(dev)
    got = buffer.to(dev)
    assert _hip.copy_pages(got, torch.tensor(pairs, dtype=torch.int32, device=dev),
                           error_flag=error) is got
    assert int(error.item()) == 0 and torch.equal(got.cpu(), expected)
    got = buffer.to(dev)
    _hip.copy_pages(got, torch.tensor(pairs + extra, dtype=torch.int32, device=dev),
                    error_flag=error)
    assert int(error.item()) == _hip.PAGED_ERANGE and torch.equal(got.cpu(), expected)
    # no pairs at all
    _hip.copy_pages(got, torch.empty((0, 2), dtype=torch.int32, device=dev))
    assert torch.equal(got.cpu(), expected)


def test_copy_pages_of_one_plane_group(gpu_device):
    # [planes, pages, bytes]: any dtype
    data = torch.arange(3 * 5 * 48, dtype=torch.int64).view(3, 5, 48)
    got = data.to(gpu_device)
    _hip.copy_pages(got, torch.tensor([[4, 1]], dtype=torch.int32, device=gpu_device))
    data[:, 1] = data[:, 4]
    assert torch.equal(got.cpu(), data)


# ------------------------------------------------------- a decode step of them


def _reference(history, q, dim):
    k = torch.stack([h[0] for h in history], 1)
    v = torch.stack([h[1] for h in history], 1)
    return attention(q, k, v, torch.ones(k.shape[1], dtype=torch.bool), dim ** -0.5)


def test_continuations_of_one_prompt(gpu_device):
    """A prompt's cache forked, each copy continued with rows of its own
    (append, attend, sample), sequences ended and the pool compacted between
    steps: every output against the sequence's own history."""

    dev, layers, kv, heads, dim, page = gpu_device, 2, 2, 8, 64, 8
    g = torch.Generator().manual_seed(21)
    prompt = SimpleKVCache(layers, kv, dim, device=dev)
    n = 21
    prompt_kv = normal((layers, 2, n, kv, dim), g)
    for layer in range(layers):
        prompt.append(layer, *(prompt_kv[layer, w].transpose(0, 1)[None].to(dev)
                               for w in (0, 1)))
    cache = PagedKVCache(40, 8, 64, layer_count=layers, num_kv_heads=kv, head_dim=dim,
                         page_size=page, device=dev)
    cache.buffer.fill_(math.nan)
    spare = cache.add()
    cache.extend([spare], 20)  # pages in front of the prompt's
    first = cache.add()
    cache.load(first, prompt)
    rows = [first] + cache.fork(first, 3)
    history = {r: [[(prompt_kv[layer, 0, p], prompt_kv[layer, 1, p]) for p in range(n)]
                   for layer in range(layers)] for r in rows}
    positions = torch.arange(64, dtype=torch.float32)[:, None]
    angle = positions * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    rope = (cos.to(dev), sin.to(dev))
    head = torch.randn(heads * dim, 301, generator=g)
    for step in range(12):
        if step == 3:
            cache.free(spare)
        if step == 5:
            cache.free(rows.pop(1))
            assert cache.compact() > 0
        if step == 8:
            new = cache.fork(rows[0])[0]
            history[new] = [list(h) for h in history[rows[0]]]
            rows.append(new)
        cache.extend(rows)
        batch = rows + [-1]  # an idle row of the batch
        at = torch.tensor([cache.length(r) - 1 for r in rows] + [-1], dtype=torch.int32)
        at_d = at.to(dev)
        rows_d = torch.tensor(batch, dtype=torch.int32, device=dev)
        for layer in range(layers):
            fused = normal((len(batch), heads + 2 * kv, dim), g)
            f = fused.to(dev)
            q_out = torch.empty(len(batch), heads, dim, dtype=torch.bfloat16, device=dev)
            out = torch.zeros_like(q_out)
            cache.append(layer, f[:, :heads], f[:, heads:heads + kv], f[:, heads + kv:],
                         at_d, rows=rows_d, rope=rope, q_out=q_out)
            cache.attend(layer, q_out, out, rows=rows_d)
            for b, r in enumerate(rows):
                page_id = cache.pages(r)[int(at[b]) // page]
                k_row = cache.k_pages(layer)[page_id, :, int(at[b]) % page].cpu()
                k_ref, k_tol = rotated(fused[b, heads:heads + kv], cos[int(at[b])],
                                       sin[int(at[b])], False)
                assert bool(((k_row.double() - k_ref).abs() <= k_tol).all())
                history[r][layer].append((k_row, fused[b, heads + kv:]))
                ref, tol = _reference(history[r][layer], q_out[b].cpu(), dim)
                assert bool(((out[b].cpu().double() - ref).abs() <= tol).all()), (step, layer, r)
        cache.check()
        logits = (out[:len(rows)].float().view(len(rows), -1).cpu() @ head).to(dev)
        ids = torch.empty(len(rows), dtype=torch.int64, device=dev)
        ws = torch.empty(_hip.sample_workspace_bytes(len(rows), 301), dtype=torch.uint8,
                         device=dev)
        _hip.sample(logits, torch.rand(len(rows), generator=g).to(dev), ids, ws,
                    temperature=0.0)
        assert torch.equal(ids, logits.argmax(-1))
    for r in rows:
        cache.free(r)
    assert cache.free_pages == cache.num_pages


def test_captured_step_replays(gpu_device):
    """append + attend + sample captured once; the cache grows between
    replays, and every replay equals the eager step."""

    dev, kv, heads, dim, page, vocab = gpu_device, 2, 8, 128, 16, 1000
    g = torch.Generator().manual_seed(31)
    cache = PagedKVCache(64, 4, 400, layer_count=1, num_kv_heads=kv, head_dim=dim,
                         page_size=page, device=dev)
    cache.buffer.zero_()
    rows = [cache.add() for _ in range(3)]
    rows_d = torch.tensor(rows, dtype=torch.int32, device=dev)
    cache.extend(rows, 250)
    cache.buffer.copy_(normal(cache.buffer.shape, g).to(dev))
    at = torch.zeros(3, dtype=torch.int32, device=dev)
    fused = torch.zeros(3, heads + 2 * kv, dim, dtype=torch.bfloat16, device=dev)
    q_out, out = (torch.zeros(3, heads, dim, dtype=torch.bfloat16, device=dev)
                  for _ in range(2))
    logits = torch.zeros(3, vocab, device=dev)
    uniform = torch.zeros(3, device=dev)
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    ws = torch.empty(_hip.sample_workspace_bytes(3, vocab), dtype=torch.uint8, device=dev)

    def step(q_out, out, ids):
        cache.append(0, fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:],
                     at, rows=rows_d, q_out=q_out)
        cache.attend(0, q_out, out, rows=rows_d)
        _hip.sample(logits, uniform, ids, ws, temperature=0.7, top_k=50, top_p=0.9,
                    min_p=0.01)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(q_out, out, ids)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q_out, out, ids)
    for replay in range(5):
        cache.extend(rows, 1 + replay)
        fused.copy_(normal(fused.shape, g).to(dev))
        logits.copy_((torch.randn(3, vocab, generator=g) * 3).to(dev))
        uniform.copy_(torch.rand(3, generator=g).to(dev))
        at.copy_(cache.lengths[rows_d.long()] - 1)
        graph.replay()
        torch.cuda.synchronize(dev)
        other = [torch.zeros_like(t) for t in (q_out, out, ids)]
        step(*other)
        torch.cuda.synchronize(dev)
        for a, b in zip((q_out, out, ids), other):
            assert torch.equal(a, b), replay
    cache.check()


def test_cache_keeps_the_device_of_its_pool():
    cache = PagedKVCache(2, 1, 16, layer_count=1, num_kv_heads=1, head_dim=64, page_size=8)
    assert cache.device == cache.buffer.device == torch.device("cuda", 0)
    assert cache.page_table.device == cache.device
    row = cache.add()
    cache.extend([row], 9)
    assert cache.page_table.tolist() == [[0, 1]] and cache.lengths.tolist() == [9]


def test_operators_on_a_stream_of_the_callers(gpu_device):
    dev = gpu_device
    pool = Pool([500, 3], 2, 64, 16, seed=41)
    q = normal((2, 4, 64), torch.Generator().manual_seed(42))
    expected, _ = attend(pool, q, None, dev)
    side = torch.cuda.Stream(dev)
    args = [t.to(dev) for t in (q, pool.k, pool.v, pool.table, pool.lengths)]
    out = torch.zeros_like(args[0])
    ws = workspace(2, 4, 2, 64, 512, dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    _hip.paged_decode_attention(*args, out, ws, 0.125, stream=side)
    side.synchronize()
    assert torch.equal(out.cpu(), expected)


@pytest.mark.parametrize("spare", [0, 2])
def test_dimensions_of_one_with_odd_strides(gpu_device, spare):
    # a stride of a dimension of one is any number: nothing may depend on it
    dev, dim = gpu_device, 64
    g = torch.Generator().manual_seed(51)
    pool = Pool([9], 1, dim, 16, seed=51, spare=spare).to(dev)
    pages = 1 + spare
    storage = normal((4096,), g).to(dev)
    q = torch.as_strided(storage, (1, 1, dim), (3, 5, 1), 512)
    k = torch.as_strided(storage, (1, 1, dim), (7, 1, 1), 1024)
    page_stride = 11 if pages == 1 else 16 * dim
    k_pages, v_pages = (torch.as_strided(p, (pages, 1, 16, dim), (page_stride, 13, dim, 1))
                        for p in (pool.k, pool.v))
    out = torch.as_strided(torch.zeros(256, dtype=torch.bfloat16, device=dev), (1, 1, dim),
                           (9, 1, 1))
    table = torch.as_strided(pool.table, (1, 1), (17, 19))
    ws = workspace(1, 1, 1, dim, 16, dev)
    _hip.paged_decode_attention(q, k_pages, v_pages, table, pool.lengths, out, ws, 0.125)
    kk, vv, good = Pool.rows_of(pool.to("cpu"), 0, 9)
    ref, tol = attention(q[0].cpu(), kk, vv, good, 0.125)
    assert bool(((out[0].cpu().double() - ref).abs() <= tol).all())
    _hip.paged_append(q, k, k, torch.tensor([9], dtype=torch.int32, device=dev), k_pages,
                      v_pages, table, q_out=out)
    assert torch.equal(k_pages[int(pool.table[0, 0]), :, 9].cpu(), k[0].cpu())
    assert torch.equal(out.cpu(), q.cpu())
    logits = torch.as_strided(torch.randn(50, generator=g).to(dev), (1, 50), (3, 1))
    ids = torch.empty(1, dtype=torch.int64, device=dev)
    ws = torch.empty(_hip.sample_workspace_bytes(1, 50), dtype=torch.uint8, device=dev)
    _hip.sample(logits, torch.zeros(1, device=dev), ids, ws, temperature=0.0)
    assert int(ids) == int(logits.argmax())
