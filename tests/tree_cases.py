"""Plain 64-bit forms of the drafted trees' operators, and the inputs their
tests share (CPU tensors)."""

import random

import torch

from paged_cases import BF16_STEP, normal


def random_parents(nodes, rng, reach=None):
    """A tree of any form; ``reach``: how far behind a node its parent may be
    (1: a chain)."""

    return [-1 if i == 0 else rng.randrange(max(0, i - (reach or i)), i)
            for i in range(nodes)]


def signed(mask):
    mask &= (1 << 64) - 1
    return mask - (1 << 64) if mask >> 63 else mask


def attention(q, k, v, seen, scale):
    """(output, tolerance) of one node: q [heads, dim], k / v [kv_heads, L,
    dim], seen [L] booleans, in 64 bits.

    Tolerance: the scores' products of bf16 values are exact in fp32 and
    their sum over dim terms is off by dim 2^-24 of the sum of magnitudes;
    the scaling, the maximum and the hardware exp2 add about 2^-21 of the
    score's magnitude and of the weight.  Weights enter the product with V off
    by at most 2^-16 of themselves, the sums over L positions round L times
    at most, each 2^-24 of the sum of magnitudes, and the result once to bf16."""

    heads, dim = q.shape
    group = heads // k.shape[0]
    out = torch.zeros(heads, dim, dtype=torch.float64)
    tol = torch.zeros(heads, dim, dtype=torch.float64)
    if not bool(seen.any()):
        return out, tol
    for g in range(k.shape[0]):
        kk, vv = k[g][seen].double(), v[g][seen].double()
        x = q[g * group:(g + 1) * group].double()
        w = torch.softmax(x @ kk.t() * scale, -1)
        magnitude = (x.abs() @ kk.abs().t()).amax(-1) * scale
        y = w @ vv
        slack = 2 * (dim * 2.0 ** -24 + 2.0 ** -21) * magnitude + 2.0 ** -19
        slack = slack + 2.0 ** -16 + 2 * kk.shape[0] * 2.0 ** -24
        heads_of = slice(g * group, (g + 1) * group)
        out[heads_of] = y
        tol[heads_of] = slack[:, None] * (w @ vv.abs()) + BF16_STEP * y.abs()
    return out, tol


class Step:
    """The rows of trees for the sequences of a Pool: ``sizes[b]`` nodes for
    table row ``rows[b]``, ``spare`` rows behind the last."""

    def __init__(self, sizes, rows, q_heads, dim, seed, spare=2, masks="tree"):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.rows, self.starts, self.parents, self.masks = list(rows), [0], [], []
        for n in sizes:
            parents = random_parents(n, rng, rng.choice((None, 1, 3)))
            mine = []
            for i, p in enumerate(parents):
                if masks == "tree":
                    mine.append((mine[p] if p >= 0 else 0) | 1 << i)
                else:  # any nodes at all; bits past the tree say nothing
                    mine.append(rng.getrandbits(64))
            self.parents += parents
            self.masks += mine
            self.starts.append(self.starts[-1] + n)
        total = self.starts[-1] + spare
        self.masks += [rng.getrandbits(64) for _ in range(spare)]
        self.q = normal((total, q_heads, dim), g, 1.5)

    def seen(self, b, node, length, good):
        """Which positions a node reads."""

        first, n = self.starts[b], self.starts[b + 1] - self.starts[b]
        seen = good.clone()
        for j in range(n):
            if not self.masks[first + node] >> j & 1:
                seen[length - n + j] = False
        return seen

    def tensors(self, device):
        """(q, starts, masks, rows) on the device."""

        return (self.q.to(device),
                torch.tensor(self.starts, dtype=torch.int32, device=device),
                torch.tensor([signed(m) for m in self.masks], dtype=torch.int64,
                             device=device),
                torch.tensor(self.rows, dtype=torch.int32, device=device))


def walk(ids, parents, targets):
    """(path, next token) of one tree's lists."""

    if not ids:
        return [], -1
    path = [0]
    while targets[path[-1]] >= 0:
        cur = path[-1]
        fits = [c for c in range(cur + 1, len(ids))
                if parents[c] == cur and ids[c] == targets[cur]]
        if not fits:
            break
        path.append(fits[0])
    return path, targets[path[-1]]
