"""Quantization to 4 bits at the ends of bf16's range and of parameters, on the
CPU."""

import pytest
import torch

from layer_streaming import W4Matrix, w4
from paged_cases import normal

BF = torch.bfloat16


def test_a_range_past_fp32_has_a_scale():
    # finite weights of both signs, 6e38 apart
    w = normal((2, 64), torch.Generator().manual_seed(1))
    w[0, 3], w[0, 40], w[0, 41] = 3e38, 3e38, -3e38
    m = W4Matrix.quantize(w, group=32, zeros=True)
    q, scales, points = m.values()
    for group, (low, high) in enumerate(((min(0.0, float(w[0, :32].min())), float(w[0, 3])),
                                         (float(w[0, 41]), float(w[0, 40])))):
        want = float(torch.tensor((high - low) / 15, dtype=torch.float64).to(BF))
        assert float(scales[0, group]) == want
        step = float(scales[0, group])
        assert int(points[0, group]) == min(15, max(0, round(-low / step)))
        for column in range(32 * group, 32 * group + 32):
            value = step * (int(q[0, column]) - int(points[0, group]))
            assert abs(value - float(w[0, column])) <= 1.01 * step
    # other groups as ever
    assert torch.equal(m.values()[1][1], W4Matrix.quantize(w[1:], group=32, zeros=True)
                       .values()[1][0])


@pytest.mark.parametrize("zeros", [False, True])
def test_a_parameter_leaves_no_graph(monkeypatch, zeros):
    w = normal((40, 64), torch.Generator().manual_seed(2))
    seen = []
    kept = w4._by_tile
    monkeypatch.setattr(w4, "_by_tile", lambda x, *sizes: (
        seen.append(x.requires_grad), kept(x, *sizes))[1])
    m = W4Matrix.quantize(torch.nn.Parameter(w), group=32, zeros=zeros)
    assert seen and not any(seen) and not m.scales.requires_grad
    for a, b in zip(m.values(), W4Matrix.quantize(w, group=32, zeros=zeros).values()):
        assert (a is None and b is None) or torch.equal(a, b)
    scales = torch.nn.Parameter(torch.ones(40, 2, dtype=BF))
    assert not W4Matrix.pack(m.values()[0], scales, group=32).scales.requires_grad
