"""Products with 4-bit weights are as near 64 bits as fp32 sums are, at the
models' sizes: the mean error, which the worst case says little of."""

import pytest
import torch

from layer_streaming import W4Matrix, _hip
from paged_cases import normal
from w4_cases import matrix, product, random_matrix, rounded
from w4_near import far, near_rounded, near_sums

pytestmark = pytest.mark.gpu

BF, U8 = torch.bfloat16, torch.uint8

# as quantized weights are: a scale of about k^-0.5 / 5
MODEL = [(4096, 14336, 64, True), (14336, 4096, 128, False), (4096, 4096, 32, True),
         (8008, 4096, 128, True), (1024, 4096, 64, False)]


def space(rows, n, k, device):
    size = _hip.linear_w4_workspace_bytes(rows, n, k)
    return torch.full((size,), 0xFF, dtype=U8, device=device)


def parts_of(n, k, group, zeros, seed, device):
    return [None if p is None else p.to(device) for p in random_matrix(n, k, group, zeros, seed)]


@pytest.mark.parametrize("n,k,group,zeros", MODEL)
@pytest.mark.parametrize("rows", [1, 5, 16, 61, 157])
def test_linear(gpu_device, rows, n, k, group, zeros):
    print("near", rows, n, k, group, zeros, flush=True)
    parts = parts_of(n, k, group, zeros, n + k, gpu_device)
    m = W4Matrix.pack(*parts, group=group)
    g = torch.Generator().manual_seed(rows)
    x, add = normal((rows, k), g).to(gpu_device), normal((rows, n), g).to(gpu_device)
    y = x.double() @ matrix(*parts, group).t()
    ws = space(rows, n, k, gpu_device)
    logits = torch.full((rows, n), 7.0, device=gpu_device)
    _hip.linear_w4(x, m, logits, workspace=ws)
    assert near_sums(logits, y), far(logits, y)
    out = torch.full((rows, n), 7.0, dtype=BF, device=gpu_device)
    _hip.linear_w4(x, m, out, workspace=ws)
    assert near_rounded(out, y), far(out, y)
    _hip.linear_w4(x, m, out, residual=add, workspace=ws)
    assert near_rounded(out, y + add.double()), far(out, y + add.double())


@pytest.mark.parametrize("rows", [1, 16, 61, 157])
@pytest.mark.parametrize("n,k,group,zeros", [(14336, 4096, 128, False), (2056, 1400, 64, True)])
def test_gate_up(gpu_device, rows, n, k, group, zeros):
    print("near gate_up", rows, n, k, group, zeros, flush=True)
    x = normal((rows, k), torch.Generator().manual_seed(rows)).to(gpu_device)
    halves, ys = [], []
    for seed in (1, 2):
        parts = parts_of(n, k, group, zeros, seed, gpu_device)
        halves.append(W4Matrix.pack(*parts, group=group))
        ys.append(x.double() @ matrix(*parts, group).t())
    out = torch.full((rows, n), 7.0, dtype=BF, device=gpu_device)
    _hip.gate_up_swiglu_w4(x, *halves, out)
    want = ys[0] * torch.sigmoid(ys[0]) * ys[1]
    assert near_rounded(out, want), far(out, want)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows", [1, 20, 70])
def test_rows_whose_terms_cancel(gpu_device, rows, zeros):
    # x of one sign, and one large entry under weights of zero: sums are of terms
    # of 24 |x| (48 |x| with zero points), and so is their rounding
    n, k, group = 200, 1024, 64
    q, scales, points = random_matrix(n, k, group, zeros, 5)
    at = 300
    q[:, at] = 8 if points is None else points[:, at // group]
    q[7] = 8 if points is None else points[7].repeat_interleave(group)  # a row of zeros
    parts = [None if p is None else p.to(gpu_device) for p in (q, scales, points)]
    m = W4Matrix.pack(*parts, group=group)
    x = normal((rows, k), torch.Generator().manual_seed(rows)).abs()
    large = x.clone()
    large[:, at] = 30000.0
    for value in (x, large):
        value = value.to(gpu_device)
        y, tol = product(value, *parts, group)
        ws = space(rows, n, k, gpu_device)
        logits = torch.full((rows, n), 7.0, device=gpu_device)
        _hip.linear_w4(value, m, logits, workspace=ws)
        assert bool(((logits.double() - y).abs() <= tol).all())
        out = torch.full((rows, n), 7.0, dtype=BF, device=gpu_device)
        _hip.linear_w4(value, m, out, workspace=ws)
        assert bool(((out.double() - y).abs() <= rounded(y, tol)).all())
        assert bool((y[:, 7] == 0).all())
