"""Plain 64-bit forms of the paged cache's operators and of sampling, and the
inputs their tests share (CPU tensors)."""

import math

import torch

BF16_STEP = 2.0 ** -8  # half a step of a rounding to bf16, relative


def normal(shape, generator, scale=1.0):
    return (torch.randn(shape, generator=generator) * scale).to(torch.bfloat16)


class Pool:
    """Page pools and a table for sequences of the given lengths, pages in
    random order, everything that no sequence holds set to NaN."""

    def __init__(self, lengths, kv_heads, dim, page_size, seed, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // page_size) for n in lengths]
        pages = sum(counts) + spare
        width = max(max(counts), 1) if width is None else width
        order = torch.randperm(pages, generator=g).tolist()
        self.k = normal((pages, kv_heads, page_size, dim), g)
        self.v = normal((pages, kv_heads, page_size, dim), g)
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        self.lengths = torch.tensor(lengths, dtype=torch.int32)
        at = 0
        for row, count in enumerate(counts):
            mine = order[at:at + count]
            at += count
            self.table[row, :count] = torch.tensor(mine, dtype=torch.int32)
            tail = lengths[row] - (count - 1) * page_size
            if count:
                self.k[mine[-1], :, tail:] = math.nan
                self.v[mine[-1], :, tail:] = math.nan
        for page in order[at:]:
            self.k[page] = math.nan
            self.v[page] = math.nan

    def to(self, device):
        for name in ("k", "v", "table", "lengths"):
            setattr(self, name, getattr(self, name).to(device))
        return self

    def rows_of(self, row, length):
        """(K, V) of a sequence as [kv_heads, length, dim], and which
        positions sit on a page of the pool."""

        page_size = self.k.shape[2]
        pages = self.table[row, :-(-length // page_size)].long()
        good = (pages >= 0) & (pages < self.k.shape[0])
        at = torch.where(good, pages, 0)

        def flat(pool):
            x = pool[at].permute(1, 0, 2, 3)
            return x.reshape(x.shape[0], -1, x.shape[3])[:, :length]

        return flat(self.k), flat(self.v), good.repeat_interleave(page_size)[:length]


def attention(q, k, v, good, scale):
    """(output, tolerance) of one token: q [heads, dim], k / v [kv_heads, L,
    dim], in 64 bits.

    Tolerance: the scores' products of bf16 values are exact in fp32 and
    their sum over dim terms is off by dim 2^-24 of the sum of magnitudes;
    the scaling, the maximum and the hardware exp2 add about 2^-21 of the
    score's magnitude and of the weight.  Each weight is rounded to bf16 for
    the product with V (half a step of its share of sum w |v|) and the result
    once more."""

    heads, dim = q.shape
    group = heads // k.shape[0]
    out = torch.zeros(heads, dim, dtype=torch.float64)
    tol = torch.zeros(heads, dim, dtype=torch.float64)
    if not bool(good.any()):
        return out, tol
    for h in range(heads):
        kk, vv = k[h // group][good].double(), v[h // group][good].double()
        x = q[h].double()
        score = kk @ x * scale
        magnitude = float((kk.abs() @ x.abs()).max()) * scale
        w = torch.softmax(score, 0)
        out[h] = w @ vv
        slack = 2 * (dim * 2.0 ** -24 + 2.0 ** -21) * magnitude + 2.0 ** -19
        spread = w @ vv.abs()
        tol[h] = (BF16_STEP + slack) * spread + BF16_STEP * out[h].abs()
    return out, tol


def rotated(x, cos, sin, interleaved):
    """(rotated, tolerance) of rows x [.., heads, dim] with cos / sin [..,
    r / 2]: three fp32 roundings of the products' magnitude, then one to
    bf16."""

    x = x.double()
    if cos is None:
        return x, torch.zeros_like(x)
    half = cos.shape[-1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    cos, sin = cos.double()[..., None, :], sin.double()[..., None, :]
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    for one, other in ((a, b), (b, a)):
        size = (x[..., one] * cos).abs() + (x[..., other] * sin).abs()
        tol[..., one] = 3 * 2.0 ** -24 * size + BF16_STEP * y[..., one].abs()
    return y, tol


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability, weight of the token) of one row, in 64 bits;
    weights are relative to the largest.

    The operator defines a weight as a multiple of 2^-44 of the largest, so
    one below 2^-45 is 0: with uniform = 0, which takes the first token of any
    weight at all, exp() alone would name a token of weight 1e-305."""

    x = logits.double()
    if bool(x.isnan().any()) or float(x.max()) == -math.inf:
        return -1, math.nan, 1.0
    top = float(x.max())
    if not temperature > 0:
        return int((x == top).nonzero()[0]), 0.0, 1.0
    w = torch.where(x == top, 1.0, ((x - top) / temperature).exp())
    w = torch.where((x == -math.inf) | (w < 2.0 ** -45), 0.0, w)
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        need, total, kept = top_p * math.fsum(float(w[i]) for i in order), 0.0, []
        for i in order:
            if kept and total >= need:
                break
            kept.append(i)
            total += float(w[i])
        order = kept
    order = sorted(i for n, i in enumerate(order) if n == 0 or float(w[i]) >= min_p)
    total = math.fsum(float(w[i]) for i in order)
    u = min(max(float(uniform), 0.0), math.nextafter(1.0, 0.0))
    seen = 0.0
    for i in order:
        seen += float(w[i])
        if seen > u * total and float(w[i]) > 0:
            break
    return i, math.log(float(w[i]) / total), float(w[i])
