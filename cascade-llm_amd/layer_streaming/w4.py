"""Matrices of 4-bit weights in the layout that the kernels read.

The reference's weights are bf16 (layer_streaming/plan.py:219-243).  A W4Matrix
holds a matrix as 4-bit values with a bf16 scale, and where wanted a zero
point, for every ``group`` consecutive columns of a row:

    W[i, k] = scale[i, k / group] * (q[i, k] - zero[i, k / group])

It is laid out once, when the weights are loaded; ``linear_w4`` and
``gate_up_swiglu_w4`` multiply by it.
"""

import operator

import torch

__all__ = ["W4Matrix"]

_PIECE = 1 << 24  # values that a layout step takes at a time


class W4Matrix:
    """A matrix [n, k] of 4-bit weights, as ``pack`` or ``quantize`` make it.

    ``packed`` (uint8), ``scales`` (bf16) and ``zeros`` (uint8, or None for a
    zero point of 8 everywhere) are in the kernels' tiles (cascade_hip.h, "4-bit
    weights"); ``values`` gives the matrix back.  The three are views of the
    matrix's memory: writing to them changes it, giving them other memory
    (``set_``, ``.data =``) does not.  Where that memory's storage is resized to
    nothing, the products refuse the matrix until it is back."""

    def __init__(self, packed, scales, zeros, n, k, group):
        n, k = operator.index(n), operator.index(k)
        group, groups = _groups(n, k, group)
        if not isinstance(packed, torch.Tensor):
            raise TypeError("packed must be a torch.Tensor")
        tiles = -(-n // 16)
        for name, part, dtype, shape in (
                ("packed", packed, torch.uint8, (tiles * -(-k // 128) * 1024,)),
                ("scales", scales, torch.bfloat16, (tiles, groups, 16)),
                ("zeros", zeros, torch.uint8, (tiles, groups, 16))):
            if part is None and name == "zeros":
                continue
            _like(packed, part, name, dtype, shape)
            if not part.is_contiguous() or part.data_ptr() % 16:
                raise ValueError("{} must be contiguous and 16-byte aligned".format(name))
        # views that nobody else can give other memory
        self._parts = tuple(None if part is None else part.detach()
                            for part in (packed, scales, zeros))
        self._sizes = n, k, group
        self._index = packed.get_device()
        # their storages; the place of each in its own, and what that has to hold
        self._storages = [None if part is None else part.untyped_storage()
                          for part in self._parts]
        self._places = []
        for part in self._parts:
            place = 0 if part is None else part.storage_offset() * part.element_size()
            end = 0 if part is None else place + part.numel() * part.element_size()
            self._places += [place, end]

    def __reduce__(self):  # a copy's addresses are its own
        return W4Matrix, (*self._parts, *self._sizes)

    def _view(self, i):
        return None if self._parts[i] is None else self._parts[i].detach()

    packed = property(lambda self: self._view(0))
    scales = property(lambda self: self._view(1))
    zeros = property(lambda self: self._view(2))
    n = property(lambda self: self._sizes[0])
    k = property(lambda self: self._sizes[1])
    group = property(lambda self: self._sizes[2])

    @property
    def launch(self):
        """What a launch takes of it: device index, addresses, sizes."""

        p, s, z = self._storages
        p_at, p_end, s_at, s_end, z_at, z_end = self._places
        if (p.nbytes() < p_end or s.nbytes() < s_end
                or (z is not None and z.nbytes() < z_end)):
            raise ValueError("the memory of the matrix was released")
        return (self._index, p.data_ptr() + p_at, s.data_ptr() + s_at,
                0 if z is None else z.data_ptr() + z_at, *self._sizes)

    @classmethod
    @torch.no_grad()
    def pack(cls, values, scales, zeros=None, group=128):
        """Lay out ``values`` (uint8 [n, k], 0..15) with ``scales`` (bf16 [n,
        ceil(k / group)]) and ``zeros`` (uint8, alike, 0..15); k a multiple of
        8, ``group`` 32, 64 or 128.  The device is that of ``values``."""

        n, k, group, groups = _sizes(values, "values", torch.uint8, group)
        _like(values, scales, "scales", torch.bfloat16, (n, groups))
        if zeros is not None:
            _like(values, zeros, "zeros", torch.uint8, (n, groups))
            if bool((zeros > 15).any()):
                raise ValueError("zeros are integers of 0 to 15")
        return cls(_tiles(values, n, k), _by_tile(scales, n, groups),
                   None if zeros is None else _by_tile(zeros, n, groups), n, k, group)

    @classmethod
    @torch.no_grad()
    def quantize(cls, weight, group=128, zeros=False):
        """4-bit weights of a bf16 matrix [n, k]: of each group's values w,

            scale = bf16(max |w| / 7), q = rint(w / scale) + 8

        or, with ``zeros``, over the range from lo = min(w, 0) to hi = max(w, 0),

            scale = bf16((hi - lo) / 15), zero = rint(-lo / scale),
            q = rint(w / scale) + zero

        in fp32, halves to even, q and zero cut to 0..15.  A group of zeros has
        scale 0; one that holds an infinity or a NaN, a NaN scale."""

        n, k, group, groups = _sizes(weight, "weight", torch.bfloat16, group)
        packed, kept, points = [], [], []
        # whole tiles of rows
        step = max(1, _PIECE // k // 16) * 16
        for start in range(0, n, step):
            w = weight[start:start + step].float()
            w = torch.nn.functional.pad(w, (0, groups * group - k))
            w = w.view(-1, groups, group)
            low = w.amin(-1, keepdim=True)
            high = w.amax(-1, keepdim=True)
            if zeros:
                low, high = low.clamp(max=0), high.clamp(min=0)
                scale = (high - low) / 15
                # (two halves of a range that fp32 does not hold)
                scale = torch.where(scale.isfinite(), scale, high / 15 - low / 15)
            else:
                scale = torch.maximum(high, -low) / 7
            scale = scale.to(torch.bfloat16).float()
            scale = torch.where(scale.isfinite(), scale, float("nan"))
            by = torch.where(scale > 0, scale, 1.0)
            zero = (-low / by).round().clamp(0, 15) if zeros else 8.0
            if zeros:
                zero = torch.where(zero.isnan(), 0.0, zero)
                points.append(zero[..., 0].to(torch.uint8))
            q = ((w / by).round() + zero).clamp(0, 15)
            q = torch.where(q.isnan() | scale.isnan(), 0.0, q).to(torch.uint8)
            packed.append(_tiles(q.view(-1, groups * group)[:, :k], q.shape[0], k))
            kept.append(scale[..., 0].to(torch.bfloat16))
        return cls(torch.cat(packed), _by_tile(torch.cat(kept), n, groups),
                   _by_tile(torch.cat(points), n, groups) if zeros else None, n, k, group)

    @property
    def device(self):
        return self.packed.device

    def nbytes(self):
        parts = (self.packed, self.scales, self.zeros)
        return sum(p.numel() * p.element_size() for p in parts if p is not None)

    def to(self, device):
        """The matrix on another device (itself where it is there)."""

        return W4Matrix(self.packed.to(device), self.scales.to(device),
                        None if self.zeros is None else self.zeros.to(device), self.n,
                        self.k, self.group)

    def values(self):
        """(q uint8 [n, k], scales bf16 [n, groups], zeros uint8 or None) as
        ``pack`` takes them."""

        tiles = -(-self.k // 128)
        words = self.packed.view(torch.int32).view(-1, tiles, 4, 16, 4).long() & 0xFFFFFFFF
        words = words >> 3 | (words & 7) << 29
        q = torch.stack([words >> (16 * (i % 2) + 4 * (i // 2)) & 15 for i in range(8)], -1)
        # [row tile, tile, g, row, j, i] -> [row tile, row, tile, j, g, i]
        q = q.to(torch.uint8).permute(0, 3, 1, 4, 2, 5).reshape(-1, tiles * 128)

        def rows_of(x):
            if x is None:
                return None
            return x.permute(0, 2, 1).reshape(-1, x.shape[1])[:self.n].contiguous()

        return q[:self.n, :self.k].contiguous(), rows_of(self.scales), rows_of(self.zeros)


def _sizes(tensor, name, dtype, group):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("{} must be a torch.Tensor".format(name))
    if tensor.dtype != dtype:
        raise TypeError("{} must be {}, got {}".format(name, dtype, tensor.dtype))
    if tensor.dim() != 2 or 0 in tensor.shape:
        raise ValueError("{} must be [n, k]".format(name))
    n, k = tensor.shape
    return (n, k, *_groups(n, k, group))


def _groups(n, k, group):
    """(group, groups of a row)."""

    group = operator.index(group)
    if group not in (32, 64, 128):
        raise ValueError("a group is 32, 64 or 128 columns, not {}".format(group))
    if n < 1 or k < 8 or k % 8:
        raise ValueError("a matrix has rows, and columns by eights: [{}, {}]".format(n, k))
    return group, -(-k // group)


def _like(values, tensor, name, dtype, shape):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("{} must be a torch.Tensor".format(name))
    if tensor.dtype != dtype:
        raise TypeError("{} must be {}, got {}".format(name, dtype, tensor.dtype))
    if tuple(tensor.shape) != shape:
        raise ValueError("{} has shape {}, expected {}".format(
            name, tuple(tensor.shape), shape))
    if tensor.device != values.device:
        raise ValueError("{} must live on {}, got {}".format(
            name, values.device, tensor.device))


def _tiles(q, n, k):
    """uint8 [n, k] as packed tiles of 16 rows and 128 columns."""

    tiles = -(-k // 128)
    out = []
    step = max(1, _PIECE // (tiles * 128) // 16) * 16
    for start in range(0, n, step):
        part = q[start:start + step]
        if bool((part > 15).any()):
            raise ValueError("values are integers of 0 to 15")
        part = torch.nn.functional.pad(part, (0, tiles * 128 - k, 0, -part.shape[0] % 16))
        # [row tile, row, tile, j, g, i] -> [row tile, tile, g, row, j, i]
        part = part.view(-1, 16, tiles, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
        words = torch.zeros(part.shape[:-1], dtype=torch.int64, device=q.device)
        for i in range(8):
            words |= part[..., i].long() << (16 * (i % 2) + 4 * (i // 2))
        words = (words << 3 | words >> 29) & 0xFFFFFFFF
        words = torch.where(words >> 31 > 0, words - (1 << 32), words).to(torch.int32)
        out.append(words.contiguous().view(torch.uint8).view(-1))
    return out[0] if len(out) == 1 else torch.cat(out)


def _by_tile(x, n, groups):
    """[n, groups] as [row tile, group, row], zeros behind row n."""

    x = torch.nn.functional.pad(x, (0, 0, 0, -n % 16))
    return x.view(-1, 16, groups).permute(0, 2, 1).contiguous()
