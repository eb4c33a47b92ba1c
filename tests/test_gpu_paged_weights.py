"""The paged attention's weights enter their product with V without a
rounding that shows: inputs whose values cancel, against the 64-bit form."""

import pytest
import torch

from layer_streaming import _hip
from paged_cases import BF16_STEP, Pool, normal

pytestmark = pytest.mark.gpu


def exact(q, k, v, scale):
    """(output, tolerance) of one sequence: q [heads, dim], k / v [kv_heads, L,
    dim], in 64 bits.

    Tolerance: the scores' fp32 sums are off by dim 2^-24 of their magnitudes,
    scaling, maximum and the hardware exp2 by about 2^-21 of the score's
    magnitude and 2^-20 of the weight, numerator and denominator alike.  A
    weight is held as two bf16 values, whose sum is off by half a step of
    half a step (2^-16 of it), and the two fp32 sums of L + 64 terms (the rows,
    their runs and waves) by (L + 64) 2^-24 each.  The result is rounded
    once."""

    group = q.shape[0] // k.shape[0]
    out, tol = [], []
    for h in range(q.shape[0]):
        kk, vv, x = k[h // group].double(), v[h // group].double(), q[h].double()
        magnitude = float((kk.abs() @ x.abs()).max()) * scale
        w = torch.softmax(kk @ x * scale, 0)
        out.append(w @ vv)
        slack = 2 * (q.shape[1] * 2.0 ** -24 + 2.0 ** -21) * magnitude + 2.0 ** -19
        slack += 2.0 ** -16 + 2 * (k.shape[1] + 64) * 2.0 ** -24
        tol.append(slack * (w @ vv.abs()) + BF16_STEP * out[-1].abs())
    return torch.stack(out), torch.stack(tol)


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(32, 8, 128), (12, 4, 64), (16, 1, 64)])
@pytest.mark.parametrize("limit", [512, 4096])  # whole rows, and runs
def test_weights_are_not_rounded_to_bf16(gpu_device, q_heads, kv_heads, dim, limit):
    print("weights", q_heads, kv_heads, dim, limit, flush=True)
    dev, page_size = gpu_device, 16
    lengths = [2, 4, 16, 34, 130, 512] + ([1100] if limit > 512 else [])
    pool = Pool(lengths, kv_heads, dim, page_size, seed=dim + limit,
                width=limit // page_size)
    # each second row of V is the one before with the other sign, and the
    # scores are small: only differences of the weights are left
    pool.v[:, :, 1::2] = -pool.v[:, :, 0::2]
    q = normal((len(lengths), q_heads, dim), torch.Generator().manual_seed(61), 0.3)
    out = torch.zeros_like(q).to(dev)
    size = _hip.paged_attention_workspace_bytes(len(lengths), q_heads, kv_heads, dim, limit)
    _hip.paged_decode_attention(
        q.to(dev), pool.k.to(dev), pool.v.to(dev), pool.table.to(dev),
        pool.lengths.to(dev), out, torch.empty(size, dtype=torch.uint8, device=dev),
        dim ** -0.5, max_length=limit)
    for row, length in enumerate(lengths):
        k, v, _ = pool.rows_of(row, length)
        ref, tol = exact(q[row], k, v, dim ** -0.5)
        off = (out[row].cpu().double() - ref).abs()
        assert bool((off <= tol).all()), (row, length, float((off / tol).max()))


def test_infinite_values_of_exact_weights(gpu_device):
    # weights that one bf16 value holds (1, 1/2, 1/4): no part of them is zero
    # or negative, which would turn the infinity into a NaN
    dev, dim = gpu_device, 64
    for length in (1, 2, 4):
        pool = Pool([length], 2, dim, 16, seed=length)
        pool.k[:] = 0.0  # equal scores
        page = int(pool.table[0, 0])
        pool.v[page, 0, length - 1, 3] = float("inf")
        pool.v[page, 1, 0, 5] = -float("inf")
        q = normal((1, 8, dim), torch.Generator().manual_seed(62))
        out = torch.zeros_like(q).to(dev)
        ws = torch.empty(_hip.paged_attention_workspace_bytes(1, 8, 2, dim, 16),
                         dtype=torch.uint8, device=dev)
        _hip.paged_decode_attention(q.to(dev), pool.k.to(dev), pool.v.to(dev),
                                    pool.table.to(dev), pool.lengths.to(dev), out, ws, 0.125)
        out = out[0].cpu()
        assert bool((out[:4, 3] == float("inf")).all())
        assert bool((out[4:, 5] == -float("inf")).all())
        out[:4, 3], out[4:, 5] = 0.0, 0.0
        assert bool(out.isfinite().all())
