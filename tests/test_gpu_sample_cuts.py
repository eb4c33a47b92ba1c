"""Cuts of a long top-k and a top-p whose borders lie far apart, against the
plain 64-bit form."""

import math

import pytest
import torch

from test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,sigma", [(4096, 1.0), (16384, 1.0), (30000, 1.5)])
@pytest.mark.parametrize("leaders", [2, 3, 6, 8])
def test_top_p_among_the_leaders_of_a_long_top_k(gpu_device, vocab, sigma, leaders):
    # a few equal logits (the odd row: nearly equal ones) with about half the
    # mass over a broad tail: P ends among them, K far below, and the bins
    # between the two ends are not listed
    print("sample", vocab, leaders, flush=True)
    g = torch.Generator().manual_seed(vocab + leaders)
    rows = 8
    base = torch.randn(1, vocab, generator=g).double() * sigma
    tail = float(base.exp().sum())
    logits = base.float().repeat(rows, 1)
    at = torch.randperm(vocab, generator=g)[:leaders]
    logits[:, at] = math.log(tail / leaders)
    logits[1::2, at] += torch.rand(leaders, generator=g) * 0.003
    # uniforms over the row, so that a cut one token short or long shows
    uniform = (torch.arange(rows) + 0.5) / rows
    uniform[-1] = 1.0 - 2.0 ** -24
    for top_k in (1025, 2000, 5000):
        if top_k >= vocab:
            continue
        for top_p in (0.1, 0.3, 0.45, 0.5, 0.55, 0.7, 0.95):
            check(logits, uniform, gpu_device, top_k=top_k, top_p=top_p)
    check(logits, uniform, gpu_device, top_k=2000, min_p=0.001,
          top_p=torch.linspace(0.2, 0.9, rows))


def test_the_cut_of_a_whole_vocabulary(gpu_device):
    g = torch.Generator().manual_seed(90)
    logits = torch.randn(3, 128256, generator=g) * 2.2
    logits[:, torch.randperm(128256, generator=g)[:3]] = 13.8
    for top_p in (0.2, 0.3, 0.4):
        check(logits, torch.tensor([0.2, 0.6, 0.95]), gpu_device, top_k=5000, top_p=top_p)
