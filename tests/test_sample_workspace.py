"""A workspace sized for the largest call serves every smaller one, on the
CPU."""

import pytest

from layer_streaming import _hip


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 16, 43, 64, 256, 300])
def test_fewer_logits_never_need_more(rows):
    # fewer logits may be cut into more chunks: the lengths around the borders
    # between chunks of 2048, 4096, 6144 and 8192, and others
    most = 1 << 19
    want = -(-256 // min(rows, 256))
    lengths = {1, 16384, 16385, most} | set(range(16500, most, 4999))
    for chunk in (2048, 4096, 6144, 8192):
        lengths |= {n for n in range(want * chunk - 1, want * chunk + 2) if 1 <= n <= most}
    needs = [_hip.sample_workspace_bytes(rows, n) for n in sorted(lengths)]
    assert needs == sorted(needs)
