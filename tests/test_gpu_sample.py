"""Sampling against its plain 64-bit form: the same token for every setting,
and its log-probability; ties, masks, infinities, NaN, settings per row, and
row lengths around the kernel's tiles."""

import math

import pytest
import torch

from layer_streaming import _hip
from paged_cases import sample as plain

pytestmark = pytest.mark.gpu


def draw(logits, uniform, device, **settings):
    rows, vocab = logits.shape
    ids = torch.full((rows,), -9, dtype=torch.int64, device=device)
    logprobs = torch.full((rows,), 9.0, device=device)
    ws = torch.full((_hip.sample_workspace_bytes(rows, vocab),), 0xFF, dtype=torch.uint8,
                    device=device)
    placed = {k: v.to(device) if isinstance(v, torch.Tensor) else v
              for k, v in settings.items()}
    got = _hip.sample(logits.to(device), uniform.to(device), ids, ws, logprobs=logprobs,
                      **placed)
    assert got is ids
    torch.cuda.synchronize(device)
    return ids.cpu(), logprobs.cpu()


def check(logits, uniform, device, **settings):
    ids, logprobs = draw(logits, uniform, device, **settings)
    for r in range(logits.shape[0]):
        mine = {k: v[r].item() if isinstance(v, torch.Tensor) else v
                for k, v in settings.items()}
        token, logprob, weight = plain(logits[r], uniform[r], **mine)
        assert int(ids[r]) == token, (r, mine, int(ids[r]), token)
        got = float(logprobs[r])
        if math.isnan(logprob):
            assert math.isnan(got)
            continue
        # one rounding to fp32; weights are multiples of 2^-44 of the largest
        # (half a step of the token's own, and of each of the sum's)
        tol = 2.0 ** -24 * abs(logprob) + 2.0 ** -45 / weight + logits.shape[1] * 2.0 ** -45
        assert abs(got - logprob) <= tol, (r, mine, got, logprob)


SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=100000),
            dict(top_p=0.0), dict(top_p=0.4), dict(top_p=0.999), dict(min_p=0.05),
            dict(min_p=1.0), dict(min_p=7.0), dict(temperature=0.3, top_k=40, top_p=0.9),
            dict(temperature=1.7, top_k=200, top_p=0.7, min_p=0.02),
            dict(temperature=0.01), dict(temperature=100.0, top_p=0.5),
            dict(temperature=2.0, top_k=700, top_p=0.99)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 1025, 8193])
def test_settings(gpu_device, vocab, settings):
    print("sample", vocab, settings, flush=True)
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(4, vocab, generator=g) * 3
    uniform = torch.tensor([0.0, 0.3, 0.77, 1.0 - 2.0 ** -24])
    check(logits, uniform, gpu_device, **settings)


@pytest.mark.parametrize("settings", SETTINGS[2:], ids=str)
def test_ties(gpu_device, settings):
    # few distinct values, both zeros, runs of one value over many tiles
    g = torch.Generator().manual_seed(7)
    logits = (torch.randn(5, 5000, generator=g) * 2).round() / 2
    logits[0, logits[0] == 0] = -0.0
    logits[1] = 0.25
    logits[2, 10:] = -3.0
    logits[3, ::2] = -math.inf
    check(logits, torch.rand(5, generator=g), gpu_device, **settings)


def test_masks_infinities_and_nan(gpu_device):
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(9, 3000, generator=g) * 4
    low = torch.finfo(torch.float32).min
    logits[0] = -math.inf                      # nothing left
    logits[1, :] = -math.inf
    logits[1, 1234] = -50.0                    # one token left
    logits[2] = low                            # all at the type's lowest value
    logits[3, 1:] = low
    logits[4, 77] = math.nan
    logits[5, [5, 900]] = math.inf             # two certain tokens
    logits[6, :2999] = -math.inf
    logits[7, 100:] = -math.inf
    logits[8] *= 1e30
    uniform = torch.tensor([0.1, 0.9, 0.5, 0.999, 0.2, 0.7, 0.0, 0.6, 0.4])
    for settings in (dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5),
                     dict(temperature=0.0), dict(temperature=0.5, top_k=50, top_p=0.9)):
        check(logits, uniform, gpu_device, **settings)
    ids, logprobs = draw(logits, uniform, gpu_device)
    assert ids[0] == -1 and ids[4] == -1
    assert math.isnan(float(logprobs[0])) and math.isnan(float(logprobs[4]))


def test_uniform_outside_is_taken_as_the_nearest_inside(gpu_device):
    logits = torch.randn(5, 400, generator=torch.Generator().manual_seed(9))
    uniform = torch.tensor([-1.0, 1.0, 5.0, math.inf, math.nan])
    ids, _ = draw(logits, uniform, gpu_device)
    assert ids.tolist() == [0, 399, 399, 399, 0]


def test_top_k_past_64_bits_is_off(gpu_device):
    g = torch.Generator().manual_seed(19)
    logits, uniform = torch.randn(8, 500, generator=g), torch.rand(8, generator=g)
    off = draw(logits, uniform, gpu_device)
    assert len(set(off[0].tolist())) > 1
    for top_k in (1 << 40, (1 << 64) + 1, -1, 1 - (1 << 64)):
        assert torch.equal(draw(logits, uniform, gpu_device, top_k=top_k)[0], off[0])


def test_settings_per_row(gpu_device):
    g = torch.Generator().manual_seed(10)
    rows, vocab = 23, 4097
    logits = torch.randn(rows, vocab, generator=g) * 2.5
    settings = dict(
        temperature=torch.where(torch.rand(rows, generator=g) < 0.2, 0.0,
                                0.2 + torch.rand(rows, generator=g)),
        top_k=torch.randint(-1, 60, (rows,), generator=g, dtype=torch.int32),
        top_p=0.2 + torch.rand(rows, generator=g), min_p=torch.rand(rows, generator=g) * 0.1)
    check(logits, torch.rand(rows, generator=g), gpu_device, **settings)
    # and mixed with one number for all
    settings["temperature"] = 0.9
    settings["top_k"] = 0
    check(logits, torch.rand(rows, generator=g), gpu_device, **settings)


@pytest.mark.parametrize("vocab", [32000, 128256])
def test_whole_vocabularies(gpu_device, vocab):
    print("sample", vocab, flush=True)
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(3, vocab, generator=g) * 2.2
    logits[1] = logits[1].to(torch.bfloat16).float()  # many ties
    wide = torch.full((3, vocab + 5), math.nan)
    wide[:, :vocab] = logits
    uniform = torch.rand(3, generator=g)
    for settings in (dict(temperature=0.8, top_k=40, top_p=0.95), dict(), dict(top_p=0.99),
                     dict(temperature=1.5, top_k=20000, top_p=0.9, min_p=0.001)):
        check(logits, uniform, gpu_device, **settings)
        a, _ = draw(logits, uniform, gpu_device, **settings)
        ids = torch.empty(3, dtype=torch.int64, device=gpu_device)
        ws = torch.empty(_hip.sample_workspace_bytes(3, vocab), dtype=torch.uint8,
                         device=gpu_device)
        _hip.sample(wide.to(gpu_device)[:, :vocab], uniform.to(gpu_device), ids, ws,
                    **settings)
        assert torch.equal(a, ids.cpu())


@pytest.mark.parametrize("vocab", [3, 1027, 4095, 4096, 4097, 8190, 16383, 16384, 16385, 16389,
                                   18433, 40961])
def test_row_lengths_around_the_kernels_tiles(gpu_device, vocab):
    # one launch up to 16384 logits, by 256 threads up to 4096; chunks of 2048
    # beyond; the last three logits of an odd row stand alone
    print("sample", vocab, flush=True)
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(4, vocab, generator=g) * 1.5
    logits[1, -1] += 9.0
    logits[2, :-2] = -math.inf
    uniform = torch.rand(4, generator=g)
    for settings in (dict(temperature=1.3), dict(top_p=0.97), dict(top_k=1500, top_p=0.9),
                     dict(top_k=1025), dict(top_k=1024, top_p=0.999, min_p=0.001),
                     dict(temperature=0.0), dict(min_p=0.3)):
        check(logits, uniform, gpu_device, **settings)


def test_lists_of_every_length(gpu_device):
    # logits that differ by less than a bin: whole rows of candidates, sorted
    # in registers, in LDS, or (past 4096) replaced by counting
    g = torch.Generator().manual_seed(5)
    for vocab, near in ((3000, 200), (3000, 300), (6000, 600), (9000, 1100), (16000, 3000),
                        (16000, 5000), (30000, 400), (30000, 700), (30000, 1500),
                        (30000, 4000), (30000, 4200)):
        print("list of", near, "in", vocab, flush=True)
        logits = torch.randn(2, vocab, generator=g) - 20.0
        for r in range(2):
            at = torch.randperm(vocab, generator=g)[:near]
            logits[r, at] = 1.0 + torch.rand(near, generator=g) * 0.004
        uniform = torch.rand(2, generator=g)
        for settings in (dict(top_p=0.6), dict(top_k=near // 2), dict(top_k=near - 1, top_p=0.7),
                         dict(top_k=torch.tensor([near // 3, 7], dtype=torch.int32),
                              top_p=0.5)):
            check(logits, uniform, gpu_device, **settings)


@pytest.mark.parametrize("vocab,equal", [(6000, 5000), (30000, 5000), (30000, 30000)])
def test_cuts_among_more_equals_than_a_list_holds(gpu_device, vocab, equal):
    # both cuts end among the same equal logits: top-p's must not bring back
    # those that top-k left out
    print("sample", equal, "equal of", vocab, flush=True)
    g = torch.Generator().manual_seed(equal + vocab)
    logits = torch.randn(4, vocab, generator=g) - 20.0
    for r in range(4):
        logits[r, torch.randperm(vocab, generator=g)[:equal]] = 1.0
    uniform = torch.rand(4, generator=g)
    for settings in (dict(top_k=1, top_p=0.95), dict(top_k=2000, top_p=0.9999999),
                     dict(top_k=2000, top_p=0.3), dict(top_k=4500, top_p=0.5, min_p=0.5)):
        check(logits, uniform, gpu_device, **settings)


@pytest.mark.parametrize("vocab", [16385, 20002, 128256, 1 << 19])
def test_short_top_k_of_long_rows(gpu_device, vocab):
    # one top_k of at most 112: lists of the chunks' largest, more than 64 of
    # them for the longest rows; 113 takes the other way
    print("sample", vocab, flush=True)
    g = torch.Generator().manual_seed(vocab + 1)
    logits = torch.randn(6, vocab, generator=g) * 2.5
    logits[1] = logits[1].to(torch.bfloat16).float()  # many ties
    logits[2, :-5] = -math.inf                        # fewer tokens than top_k
    logits[3, 2048:] = -100.0                         # one chunk has them all, and
    logits[3, 300:] -= 1000.0                         # few have a weight
    logits[4] = logits[4].clamp(max=0.0) * 0.01
    logits[4, ::7] = -0.0
    logits[5, vocab // 2] = math.inf
    uniform = torch.tensor([0.3, 0.999, 0.6, 0.0, 0.45, 0.8])
    for top_k in (1, 40, 112) if vocab > 200000 else (1, 2, 40, 55, 56, 64, 65, 112, 113):
        check(logits, uniform, gpu_device, temperature=0.8, top_k=top_k, top_p=0.95)
    for settings in (dict(top_k=100, min_p=0.2), dict(top_k=3, min_p=1.5),
                     dict(top_k=112, top_p=0.0), dict(temperature=0.0, top_k=40),
                     dict(temperature=50.0, top_k=90, top_p=0.7)):
        if vocab > 200000:  # (the plain form sorts in Python)
            break
        check(logits, uniform, gpu_device, **settings)
    temperature = torch.tensor([0.0, 1.0, 0.0, 0.5, 0.0, 2.0])
    check(logits, uniform, gpu_device, temperature=temperature, top_k=20,
          top_p=torch.tensor([0.5, 1.0, 0.1, 0.9, 1.0, 0.3]))
    logits[0, vocab - 1] = math.nan
    logits[1] = -math.inf
    ids, logprobs = draw(logits, uniform, gpu_device, top_k=7)
    assert ids[:2].tolist() == [-1, -1] and bool(logprobs[:2].isnan().all())
    assert bool((ids[2:] >= 0).all())


@pytest.mark.parametrize("vocab,near", [(30000, 100), (30000, 300), (30000, 700),
                                        (30000, 4200), (30000, 30000), (61440, 3000),
                                        (61440, 5000)])
def test_short_top_k_among_equals(gpu_device, vocab, near):
    # `near` tokens in one bin: the chunks' lists are longer than top_k, or
    # than they can be; so is the row's
    print("sample", near, "in", vocab, flush=True)
    g = torch.Generator().manual_seed(near)
    logits = torch.randn(3, vocab, generator=g) - 20.0
    for r in range(3):
        at = torch.randperm(vocab, generator=g)[:near]
        logits[r, at] = 1.0 if r == 2 else 1.0 + torch.rand(near, generator=g) * 0.004
    uniform = torch.rand(3, generator=g)
    for settings in (dict(top_k=1), dict(top_k=40), dict(top_k=112, top_p=0.6),
                     dict(top_k=99, min_p=0.9), dict(top_k=112, temperature=0.5)):
        check(logits, uniform, gpu_device, **settings)


def test_what_the_workspace_held_is_not_read(gpu_device):
    # bytes that are keys of large logits, numbers of tokens and masses; lists
    # that are written in part
    g = torch.Generator().manual_seed(78)
    for vocab, near in ((30000, 30000), (150000, 150000), (30000, 900), (9000, 5000)):
        print("sample", near, "in", vocab, flush=True)
        logits = torch.randn(2, vocab, generator=g) - 20.0
        logits[:, :near] = 1.0
        uniform = torch.rand(2, generator=g).to(gpu_device)
        on_device = logits.to(gpu_device)
        for settings in (dict(top_k=40, top_p=0.9), dict(top_k=300), dict(top_p=0.6), dict()):
            found = []
            for byte in (0, 0xC5, 0x3F, 0xFF):
                ids = torch.empty(2, dtype=torch.int64, device=gpu_device)
                ws = torch.full((_hip.sample_workspace_bytes(2, vocab),), byte,
                                dtype=torch.uint8, device=gpu_device)
                _hip.sample(on_device, uniform, ids, ws, **settings)
                found.append(ids.tolist())
            assert all(ids == found[0] for ids in found), (settings, found)


def test_captured_draws_replay(gpu_device):
    # both forms of long rows in one graph, and another graph, share a workspace
    dev, vocab = gpu_device, 50000
    g = torch.Generator().manual_seed(79)
    logits, uniform = torch.zeros(3, vocab, device=dev), torch.zeros(3, device=dev)
    ws = torch.empty(_hip.sample_workspace_bytes(3, vocab), dtype=torch.uint8, device=dev)
    forms = (dict(top_k=40, top_p=0.9), dict(top_k=500, top_p=0.95, min_p=0.01), dict())
    ids = [torch.zeros(3, dtype=torch.int64, device=dev) for _ in forms]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        _hip.sample(logits, uniform, ids[0], ws)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, which in zip(graphs, ((0, 1), (2, 0))):
        with torch.cuda.graph(graph):
            for i in which:
                _hip.sample(logits, uniform, ids[i], ws, **forms[i])
    for replay in range(4):
        logits.copy_((torch.randn(3, vocab, generator=g) * 3).to(dev))
        uniform.copy_(torch.rand(3, generator=g).to(dev))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize(dev)
        for i, form in enumerate(forms):
            eager = torch.zeros(3, dtype=torch.int64, device=dev)
            _hip.sample(logits, uniform, eager, ws, **form)
            assert torch.equal(ids[i], eager), (replay, form)


def test_short_top_k_of_many_rows(gpu_device):
    # the rows of two slices, chunks of 8192
    g = torch.Generator().manual_seed(77)
    logits, uniform = torch.randn(300, 17000, generator=g) * 3, torch.rand(300, generator=g)
    check(logits, uniform, gpu_device, temperature=0.9, top_k=40, top_p=0.9)


def test_on_a_stream_of_the_callers(gpu_device):
    g = torch.Generator().manual_seed(6)
    for vocab in (3000, 50000):
        logits = (torch.randn(3, vocab, generator=g) * 2).to(gpu_device)
        uniform = torch.rand(3, generator=g).to(gpu_device)
        ws = torch.empty(_hip.sample_workspace_bytes(3, vocab), dtype=torch.uint8,
                         device=gpu_device)
        one, other = (torch.zeros(3, dtype=torch.int64, device=gpu_device) for _ in range(2))
        _hip.sample(logits, uniform, one, ws, top_k=30, top_p=0.9)
        side = torch.cuda.Stream(gpu_device)
        side.wait_stream(torch.cuda.current_stream(gpu_device))
        _hip.sample(logits, uniform, other, ws, top_k=30, top_p=0.9, stream=side)
        side.synchronize()
        assert torch.equal(one, other)


@pytest.mark.parametrize("vocab", [900, 5000, 20000])
def test_extreme_temperatures(gpu_device, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(3, vocab, generator=g)
    uniform = torch.rand(3, generator=g)
    # the smallest numbers above 0: the largest logit, drawn with certainty
    for t in (5e-324, 1e-310, 1e-40):
        ids, logprobs = draw(logits, uniform, gpu_device, temperature=t)
        assert torch.equal(ids, logits.argmax(-1)) and bool((logprobs == 0).all())
        ids, _ = draw(logits, uniform, gpu_device, temperature=t, top_k=20, top_p=0.9)
        assert torch.equal(ids, logits.argmax(-1))
    # an infinite one: every token that is not masked alike
    logits[:, ::3] = -math.inf
    live = [i for i in range(vocab) if i % 3]
    ids, logprobs = draw(logits, uniform, gpu_device, temperature=math.inf)
    for r in range(3):
        assert int(ids[r]) == live[int(float(uniform[r]) * len(live))]
        assert abs(float(logprobs[r]) + math.log(len(live))) <= 2.0 ** -24 * math.log(len(live))


def test_rows_past_one_slice(gpu_device):
    # more rows than one launch's workspace holds, of the longer kind
    g = torch.Generator().manual_seed(77)
    rows, vocab = 300, 17000
    logits = torch.randn(rows, vocab, generator=g) * 2
    uniform = torch.rand(rows, generator=g)
    settings = dict(temperature=0.5 + torch.rand(rows, generator=g), top_k=30, top_p=0.9)
    ids, logprobs = draw(logits, uniform, gpu_device, **settings)
    for first in (0, 100, 250, 299):
        part = {k: v[first:first + 1] if isinstance(v, torch.Tensor) else v
                for k, v in settings.items()}
        one, lp = draw(logits[first:first + 1], uniform[first:first + 1], gpu_device, **part)
        assert one[0] == ids[first] and lp[0] == logprobs[first]
        mine = {k: v[0].item() if isinstance(v, torch.Tensor) else v for k, v in part.items()}
        assert int(one[0]) == plain(logits[first], uniform[first], **mine)[0]


def test_frequencies(gpu_device):
    # evenly spaced uniforms: each token's count is its probability, to one
    # draw either way
    n = 4096
    logits = torch.tensor([0.5, -1.0, 2.0, -math.inf, 1.0, 0.0, -2.0])
    uniform = (torch.arange(n) + 0.5) / n
    ids, _ = draw(logits.repeat(n, 1), uniform, gpu_device, temperature=1.3)
    p = torch.softmax(logits.double() / 1.3, 0)
    counts = torch.bincount(ids, minlength=7)
    assert bool(((counts - p * n).abs() <= 1.0).all())
