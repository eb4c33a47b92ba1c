"""Products with 4-bit weights against their plain form in 64 bits."""

import math

import pytest
import torch

from layer_streaming import W4Matrix, _hip
from paged_cases import normal
from w4_cases import matrix, product, random_matrix, rounded

pytestmark = pytest.mark.gpu

BF, U8 = torch.bfloat16, torch.uint8


def space(rows, n, k, device):
    size = _hip.linear_w4_workspace_bytes(rows, n, k)
    return torch.full((size,), 0xFF, dtype=U8, device=device)


def linear_case(device, rows, n, k, group, zeros, residual=False, logits=False, seed=0):
    """Runs one product and holds it to the bound."""

    parts = random_matrix(n, k, group, zeros, seed + n + k)
    g = torch.Generator().manual_seed(seed + rows)
    x = normal((rows, k), g)
    add = normal((rows, n), g) if residual else None
    m = W4Matrix.pack(*(None if p is None else p.to(device) for p in parts), group=group)
    out = torch.full((rows, n), 7.0, dtype=torch.float32 if logits else BF, device=device)
    got = _hip.linear_w4(x.to(device), m, out, workspace=space(rows, n, k, device),
                         residual=None if add is None else add.to(device))
    assert got is out
    y, tol = product(x.to(device), *(None if p is None else p.to(device) for p in parts), group)
    if add is not None:
        y = y + add.to(device).double()
        tol = tol + 2.0 ** -24 * y.abs()
    tol = tol if logits else rounded(y, tol)
    off = (out.double() - y).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))


SIZES = [(1, 8), (16, 64), (17, 72), (33, 128), (15, 136), (100, 1000), (257, 520),
         (1024, 4096), (4096, 1024), (130, 14336), (2000, 2056), (6144, 4096)]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", [1, 2, 5, 16, 17, 61, 64, 65, 130])
def test_linear_sizes(gpu_device, rows, n, k):
    print("linear", rows, n, k, flush=True)
    linear_case(gpu_device, rows, n, k, (32, 64, 128)[(rows + n) % 3], (rows + k // 8) % 2 == 0,
                residual=rows % 2 == 0)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,n,k", [(1, 48, 4104), (9, 300, 600), (40, 4096, 4096),
                                      (700, 500, 392)])
def test_linear_forms(gpu_device, group, zeros, rows, n, k):
    print("forms", group, zeros, rows, n, k, flush=True)
    linear_case(gpu_device, rows, n, k, group, zeros, residual=True, seed=1)
    linear_case(gpu_device, rows, n, k, group, zeros, logits=True, seed=2)
    linear_case(gpu_device, rows, n, k, group, zeros, seed=3)


@pytest.mark.parametrize("rows", [1, 7, 16, 33, 64, 100, 256])
def test_linear_of_the_models_sizes(gpu_device, rows):
    for n, k in ((4096, 14336), (14336, 4096), (1024, 4096), (8008, 4096)):
        print("model", rows, n, k, flush=True)
        linear_case(gpu_device, rows, n, k, 128, rows % 2 == 0, residual=True, seed=4)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_linear_of_many_rows(gpu_device, group, zeros):
    # workgroups of 16 rows over a short K, of 64 over a longer one
    print("many rows", group, zeros, flush=True)
    for k in (264, 520):
        linear_case(gpu_device, 1001, 4100, k, group, zeros, residual=True, seed=7)
        linear_case(gpu_device, 1001, 4100, k, group, zeros, logits=True, seed=8)


def test_linear_past_the_caches(gpu_device):
    # 128 MB and more of packed weights, read past the caches
    print("past the caches", flush=True)
    m, group, rows = 65552, 128, 3
    g = torch.Generator().manual_seed(1)
    part = random_matrix(1024, 4096, group, False, 1)
    times = -(-m // 1024)
    q = part[0].to(gpu_device).repeat(times, 1)[:m]
    # (no two of the repeated rows alike)
    scales = (part[1].to(gpu_device).repeat(times, 1)[:m].float()
              * (1 + torch.arange(m, device=gpu_device)[:, None] / 65536)).to(BF)
    x = normal((rows, 4096), g).to(gpu_device)
    matrix4 = W4Matrix.pack(q, scales, group=group)
    out = torch.full((rows, m), 7.0, device=gpu_device)
    _hip.linear_w4(x, matrix4, out, workspace=space(rows, m, 4096, gpu_device))
    y, tol = product(x, q, scales, None, group)
    off = (out.double() - y).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))


def test_a_split_product_needs_its_workspace(gpu_device):
    rows, n, k = 16, 256, 14336
    size = _hip.linear_w4_workspace_bytes(rows, n, k)
    assert size > 0
    m = W4Matrix.pack(*(p.to(gpu_device) for p in random_matrix(n, k, 64, True, 3)), group=64)
    x = normal((rows, k), torch.Generator().manual_seed(3)).to(gpu_device)
    out = torch.full((rows, n), 7.0, dtype=BF, device=gpu_device)
    for ws in (None, torch.zeros(size - 1, dtype=U8, device=gpu_device)):
        with pytest.raises(RuntimeError, match="workspace"):
            _hip.linear_w4(x, m, out, workspace=ws)
    odd = torch.zeros(size + 8, dtype=U8, device=gpu_device)[8:]
    with pytest.raises(RuntimeError, match="align"):
        _hip.linear_w4(x, m, out, workspace=odd)
    torch.cuda.synchronize(gpu_device)
    assert bool((out == 7).all())


@pytest.mark.parametrize("rows,n,k,group,zeros", [
    (157, 14336, 264, 32, False), (100, 33000, 136, 128, True),
    (157, 14336, 520, 64, True), (130, 14336, 520, 32, False), (100, 33000, 392, 128, True),
    (1, 16, 64, 32, True), (1, 14336, 4096, 128, False), (3, 100, 1000, 64, True),
    (16, 257, 264, 32, False), (17, 2000, 520, 128, True), (61, 14336, 4096, 64, True),
    (64, 48, 14336, 128, False), (65, 300, 72, 32, True), (200, 500, 1032, 64, False),
    (1, 1, 8, 128, True)])
def test_gate_up(gpu_device, rows, n, k, group, zeros):
    print("gate_up", rows, n, k, group, zeros, flush=True)
    halves, ys, tols = [], [], []
    x = normal((rows, k), torch.Generator().manual_seed(rows)).to(gpu_device)
    for seed in (1, 2):
        parts = [None if p is None else p.to(gpu_device)
                 for p in random_matrix(n, k, group, zeros, seed)]
        halves.append(W4Matrix.pack(*parts, group=group))
        y, tol = product(x, *parts, group)
        ys.append(y)
        tols.append(tol)
    out = torch.full((rows, n), 7.0, dtype=BF, device=gpu_device)
    assert _hip.gate_up_swiglu_w4(x, *halves, out) is out
    silu = ys[0] * torch.sigmoid(ys[0])
    want = silu * ys[1]
    # silu has a slope of at most 1.1; exp, the quotient and the products add
    # a few roundings, each relative, and of the exponent's own 2^-23 |gate|
    tol = (1.1 * tols[0] * (ys[1].abs() + tols[1]) + silu.abs() * tols[1]
           + (2.0 ** -20 + 2.0 ** -22 * ys[0].abs()) * want.abs())
    tol = rounded(want, tol)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))


def test_gate_far_below_zero_gives_zero_and_far_above_itself(gpu_device):
    # gate of -30000 and +30000 in one column each
    q = torch.full((16, 64), 9, dtype=U8)
    scales = torch.full((16, 2), 1.0, dtype=BF)
    m = W4Matrix.pack(q.to(gpu_device), scales.to(gpu_device), group=32)
    x = torch.tensor([[-468.75], [468.75], [0.0]]).expand(3, 64).to(BF).contiguous()
    x = x.to(gpu_device)
    out = torch.zeros(3, 16, dtype=BF, device=gpu_device)
    _hip.gate_up_swiglu_w4(x, m, m, out)
    value = float(x[1, 0]) * 64
    assert bool((out[0].float().abs() == 0).all()) and bool((out[2] == 0).all())
    assert bool(((out[1].double() - value * value).abs() <= 2.0 ** -7 * value * value).all())


def test_views(gpu_device):
    # rows of wider tensors on every side; what lies beside stays
    parts = [p.to(gpu_device) for p in random_matrix(100, 264, 64, True, 5)]
    m = W4Matrix.pack(*parts, group=64)
    g = torch.Generator().manual_seed(5)
    for rows in (1, 4, 40):
        fused = normal((rows, 400), g).to(gpu_device)
        x = fused[:, 64:328]
        wide = torch.full((rows, 311), 7.0, dtype=BF, device=gpu_device)
        add = normal((rows, 205), g).to(gpu_device)[:, 3:103]
        _hip.linear_w4(x, m, wide[:, 101:201], residual=add,
                       workspace=space(rows, 100, 264, gpu_device))
        y, tol = product(x, *parts, 64)
        y = y + add.double()
        tol = rounded(y, tol + 2.0 ** -24 * y.abs())
        assert bool(((wide[:, 101:201].double() - y).abs() <= tol).all())
        assert bool((wide[:, :101] == 7).all()) and bool((wide[:, 201:] == 7).all())
        f32 = torch.full((rows, 311), 7.0, device=gpu_device)
        _hip.linear_w4(x, m, f32[:, 11:111], workspace=space(rows, 100, 264, gpu_device))
        y, tol = product(x, *parts, 64)
        assert bool(((f32[:, 11:111].double() - y).abs() <= tol).all())
        assert bool((f32[:, :11] == 7).all()) and bool((f32[:, 111:] == 7).all())
        wide.fill_(7.0)
        _hip.gate_up_swiglu_w4(x, m, m, wide[:, 101:201])
        assert bool((wide[:, :101] == 7).all()) and bool((wide[:, 201:] == 7).all())
        assert bool((wide[:, 101:201] != 7).any())


def test_one_row_shared_by_all(gpu_device):
    # an expanded x has no row stride of its own
    parts = [p.to(gpu_device) for p in random_matrix(64, 128, 32, True, 6)]
    m = W4Matrix.pack(*parts, group=32)
    x = normal((1, 128), torch.Generator().manual_seed(6)).to(gpu_device)
    out = torch.zeros(1, 64, dtype=BF, device=gpu_device)
    _hip.linear_w4(x[:1], m, out, workspace=space(1, 64, 128, gpu_device))
    y, tol = product(x, *parts, 32)
    assert bool(((out.double() - y).abs() <= rounded(y, tol)).all())


def test_residual_in_place(gpu_device):
    for rows, n, k in ((1, 4096, 4096), (16, 4096, 14336), (61, 4096, 14336), (157, 4096, 4096)):
        m = W4Matrix.pack(*(p.to(gpu_device) for p in random_matrix(n, k, 64, True, 7)), group=64)
        g = torch.Generator().manual_seed(7)
        x, add = normal((rows, k), g).to(gpu_device), normal((rows, n), g).to(gpu_device)
        apart = torch.empty_like(add)
        ws = space(rows, n, k, gpu_device)
        _hip.linear_w4(x, m, apart, residual=add, workspace=ws)
        _hip.linear_w4(x, m, add, residual=add, workspace=ws)
        assert torch.equal(add, apart)


@pytest.mark.parametrize("rows", [3, 20, 70])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_row_of_no_numbers_keeps_to_itself(gpu_device, rows, value):
    parts = [p.to(gpu_device) for p in random_matrix(50, 264, 64, True, 8)]
    m = W4Matrix.pack(*parts, group=64)
    x = normal((rows, 264), torch.Generator().manual_seed(8)).to(gpu_device)
    ws = space(rows, 50, 264, gpu_device)
    clean = torch.zeros(rows, 50, dtype=BF, device=gpu_device)
    _hip.linear_w4(x, m, clean, workspace=ws)
    x[1, 100] = value
    out = torch.zeros_like(clean)
    _hip.linear_w4(x, m, out, workspace=ws)
    others = [r for r in range(rows) if r != 1]
    assert torch.equal(out[others], clean[others])
    # (a weight of 0 times an infinity is a NaN)
    assert not bool(out[1].isfinite().any())


def test_a_nan_scale_shows_in_its_row_only(gpu_device):
    q, scales, points = random_matrix(40, 264, 64, True, 9)
    x = normal((5, 264), torch.Generator().manual_seed(9)).to(gpu_device)
    outs = []
    for bad in (False, True):
        if bad:
            scales[21, 3] = math.nan
        m = W4Matrix.pack(q.to(gpu_device), scales.to(gpu_device),
                          zeros=points.to(gpu_device), group=64)
        out = torch.zeros(5, 40, dtype=BF, device=gpu_device)
        _hip.linear_w4(x, m, out, workspace=space(5, 40, 264, gpu_device))
        outs.append(out)
    others = [c for c in range(40) if c != 21]
    assert bool(outs[1][:, 21].isnan().all())
    assert torch.equal(outs[0][:, others], outs[1][:, others])


def test_columns_behind_the_last_are_not_read(gpu_device):
    # k ends inside a tile and a group; the row goes on with NaN
    for k in (8, 72, 136, 200, 264):
        parts = [p.to(gpu_device) for p in random_matrix(33, k, 128, True, k)]
        m = W4Matrix.pack(*parts, group=128)
        for rows in (1, 18, 80):
            wide = torch.full((rows, k + 128), math.nan, dtype=BF, device=gpu_device)
            wide[:, :k] = normal((rows, k), torch.Generator().manual_seed(k)).to(gpu_device)
            out = torch.zeros(rows, 33, dtype=BF, device=gpu_device)
            _hip.linear_w4(wide[:, :k], m, out, workspace=space(rows, 33, k, gpu_device))
            y, tol = product(wide[:, :k], *parts, 128)
            assert bool(((out.double() - y).abs() <= rounded(y, tol)).all()), (k, rows)


def test_captured_products_replay(gpu_device):
    # two graphs share the workspace; eager calls between the replays
    sizes = [(16, 4096, 14336), (1, 1024, 4096), (61, 4096, 4096)]
    cases = []
    for rows, n, k in sizes:
        m = W4Matrix.pack(*(p.to(gpu_device) for p in random_matrix(n, k, 64, True, rows)),
                          group=64)
        g = torch.Generator().manual_seed(rows)
        cases.append((normal((rows, k), g).to(gpu_device), m,
                      torch.zeros(rows, n, dtype=BF, device=gpu_device)))
    ws = torch.full((max(_hip.linear_w4_workspace_bytes(*s) for s in sizes),), 0xFF,
                    dtype=U8, device=gpu_device)

    def step():
        for x, m, out in cases:
            _hip.linear_w4(x, m, out, workspace=ws)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step()
    for replay in range(4):
        for x, _, out in cases:
            x.copy_(normal(x.shape, torch.Generator().manual_seed(50 + replay)).to(gpu_device))
            out.zero_()
        graphs[replay % 2].replay()
        torch.cuda.synchronize()
        replayed = [out.clone() for _, _, out in cases]
        step()
        torch.cuda.synchronize()
        for (_, _, out), again in zip(cases, replayed):
            assert torch.equal(out, again)


def test_another_stream(gpu_device):
    parts = [p.to(gpu_device) for p in random_matrix(4096, 14336, 128, True, 10)]
    m = W4Matrix.pack(*parts, group=128)
    x = normal((16, 14336), torch.Generator().manual_seed(10)).to(gpu_device)
    ws = space(16, 4096, 14336, gpu_device)
    outs = [torch.zeros(16, 4096, dtype=BF, device=gpu_device) for _ in range(3)]
    _hip.linear_w4(x, m, outs[0], workspace=ws)
    stream = torch.cuda.Stream(gpu_device)
    stream.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(stream):
        _hip.linear_w4(x, m, outs[1], workspace=ws)
    _hip.linear_w4(x, m, outs[2], workspace=torch.empty_like(ws), stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_feed_forward_in_four_bits(gpu_device):
    """A layer's feed-forward as a model runs it, from bf16 weights on: norm,
    gate and up, down onto the residual, for one token and for a tree's rows."""

    hidden, inner = 512, 1400
    g = torch.Generator().manual_seed(11)
    weights = {name: normal(shape, g, shape[1] ** -0.5) for name, shape in (
        ("gate", (inner, hidden)), ("up", (inner, hidden)), ("down", (hidden, inner)))}
    held = {name: W4Matrix.quantize(w.to(gpu_device), group=64, zeros=True)
            for name, w in weights.items()}
    exact = {name: matrix(*m.values(), 64) for name, m in held.items()}
    norm = normal((hidden,), g).to(gpu_device)
    for rows in (1, 13, 64):
        x = normal((rows, hidden), g).to(gpu_device)
        normed, act, out = (torch.empty(rows, w, dtype=BF, device=gpu_device)
                            for w in (hidden, inner, hidden))
        _hip.rmsnorm(x, norm, normed, 1e-5)
        _hip.gate_up_swiglu_w4(normed, held["gate"], held["up"], act)
        _hip.linear_w4(act, held["down"], out, residual=x,
                       workspace=space(rows, hidden, inner, gpu_device))
        gate, up = (normed.double() @ exact[n].t() for n in ("gate", "up"))
        want = gate * torch.sigmoid(gate) * up
        # one rounding of act, 2^-8, and sums that fp32 holds to far less
        assert bool(((act.double() - want).abs() <= 2.0 ** -7.9 * want.abs() + 1e-4).all())
        down = act.double() @ exact["down"].t() + x.double()
        size = act.double().abs() @ exact["down"].abs().t()
        assert bool(((out.double() - down).abs()
                     <= 2.0 ** -8 * down.abs() + 1e-4 * size).all())
        # four bits of weights: near what the bf16 weights give
        full = x.double() + (lambda a: a @ weights["down"].to(gpu_device).double().t())(
            (lambda a, b: a * torch.sigmoid(a) * b)(*(
                normed.double() @ weights[n].to(gpu_device).double().t()
                for n in ("gate", "up"))))
        assert float((out.double() - full).norm() / (full - x.double()).norm()) < 0.3
