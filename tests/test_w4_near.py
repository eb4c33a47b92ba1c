"""The bounds on the mean error of 4-bit products tell fp32 sums from rounded
ones, at the models' sizes and on the CPU: mistakes are planted in copies of the
plain form's operands."""

import pytest
import torch

from paged_cases import normal
from w4_cases import matrix, random_matrix
from w4_near import near_rounded, near_sums

BF = torch.bfloat16
SIZES = [(256, 4096, 128, False), (256, 4096, 128, True), (128, 14336, 64, True)]


def case(n, k, group, zeros):
    parts = random_matrix(n, k, group, zeros, n + k)
    x = normal((5, k), torch.Generator().manual_seed(k))
    w = matrix(*parts, group)
    return x, parts, w, x.double() @ w.t()


@pytest.mark.parametrize("n,k,group,zeros", SIZES)
def test_sums_of_fp32_pass(n, k, group, zeros):
    # of the plain form, and of the kernels' terms: 16 + q, or 48 + q - zero
    x, (q, scales, points), w, y = case(n, k, group, zeros)
    plain = x.float() @ w.float().t()
    groups = scales.shape[1]
    split = lambda t: torch.nn.functional.pad(t, (0, groups * group - k)).view(-1, groups, group)
    at = torch.arange(k) // group
    terms = 16 + q.float() if points is None else 48 + q.float() - points.float()[:, at]
    shift = -24.0 if points is None else -48.0
    xs, ts = split(x.float()), split(terms)
    sums = torch.einsum("rgk,ngk->rng", xs, ts) + shift * xs.sum(-1)[:, None]
    shifted = (sums * scales.float()[None]).sum(-1)
    for out in (plain, shifted):
        assert near_sums(out, y) and near_rounded(out.to(BF), y)


@pytest.mark.parametrize("n,k,group,zeros", SIZES)
def test_what_loses_bits_does_not(n, k, group, zeros):
    x, (q, scales, points), w, y = case(n, k, group, zeros)
    exact = x.double()
    rounded_logits = y.float().to(BF).float()
    rounded_weights = (exact @ w.to(BF).double().t()).float()
    flipped = q.clone()
    flipped[:, k // 3] ^= 1
    low_bit = (exact @ matrix(flipped, scales, points, group).t()).float()
    missing = exact.clone()
    missing[:, -1] = 0
    no_column = (missing @ w.t()).float()
    twice = y.float().to(BF).float() * (1 + 2.0 ** -9)
    for out in (rounded_logits, rounded_weights, low_bit, no_column, twice):
        assert not near_sums(out, y)
    # of bf16 rows: what is larger than their rounding
    other_scales = (exact @ matrix(q, scales * (1 + 2.0 ** -6), points, group).t()).float()
    for out in (other_scales, twice * (1 + 2.0 ** -9)):
        assert not near_rounded(out.to(BF), y)
