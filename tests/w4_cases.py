"""Plain 64-bit forms of the products with 4-bit weights, and the inputs their
tests share (CPU tensors)."""

import torch

from paged_cases import BF16_STEP, normal


def random_matrix(n, k, group, zeros, seed):
    """(values, scales, zeros or None) of a matrix [n, k]."""

    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    q = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = normal((n, groups), g, k ** -0.5)
    points = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8)
    return q, scales, points if zeros else None


def matrix(q, scales, zeros, group):
    """The matrix in 64 bits."""

    place = torch.arange(q.shape[1], device=q.device) // group
    zero = 8.0 if zeros is None else zeros.double()[:, place]
    return (q.double() - zero) * scales.double()[:, place]


def product(x, q, scales, zeros, group):
    """(x W^T, bound of an fp32 sum's error), in 64 bits.

    The kernels' terms are x (16 + q) and 24 x, or with zero points x (48 + q -
    zero) and 48 x: products of bf16 values that fp32 holds exactly, together of
    magnitude 55 |x| or 111 |x| at most.  A group's sum has at most 2 group such
    additions, each off by at most 2^-23 of the sum of magnitudes so far (a
    matrix instruction may cut where fp32 rounds), and the groups' products with
    their scales are summed with as many roundings as there are groups, one for
    the product, and 16 of partial sums that are joined."""

    x = x.double()
    size = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device=x.device)
    kept = torch.zeros_like(size)
    groups = scales.shape[1]
    for i in range(groups):
        part = slice(i * group, (i + 1) * group)
        total = x[:, part].abs().sum(1)[:, None]
        s = scales[:, i].double().abs()
        size += (55 if zeros is None else 111) * total * s
        kept += 16 * total * s
    y = x @ matrix(q, scales, zeros, group).t()
    return y, 2.0 ** -23 * (2 * group * size + (groups + 17) * kept)


def rounded(y, tol):
    """The bound with the result's rounding to bf16."""

    return tol + BF16_STEP * (y.abs() + tol) + 2.0 ** -134
