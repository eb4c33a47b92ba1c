"""Matrices of 4-bit weights on the CPU: their layout, their quantization, and
what the products refuse.  No kernel is launched."""

import math

import pytest
import torch

from layer_streaming import W4Matrix, _hip
from paged_cases import normal
from w4_cases import random_matrix

BF, U8 = torch.bfloat16, torch.uint8


@pytest.mark.parametrize("n,k,group,zeros", [
    (1, 8, 32, False), (16, 128, 128, True), (17, 136, 64, True), (40, 1000, 128, False),
    (33, 264, 32, True), (300, 64, 32, False)])
def test_the_layout_holds_the_matrix(n, k, group, zeros):
    q, scales, points = random_matrix(n, k, group, zeros, n + k)
    m = W4Matrix.pack(q, scales, zeros=points, group=group)
    assert (m.n, m.k, m.group) == (n, k, group) and m.device == q.device
    tiles, wide = -(-n // 16), -(-k // 128)
    assert m.packed.shape == (tiles * wide * 1024,)
    assert m.scales.shape == (tiles, -(-k // group), 16)
    got = m.values()
    assert torch.equal(got[0], q) and torch.equal(got[1], scales)
    assert got[2] is None if points is None else torch.equal(got[2], points)
    # a few values by the layout's description in the header
    words = m.packed.view(torch.int32)
    for row, col in ((0, 0), (n - 1, k - 1), (n // 2, k // 2), (0, k - 1), (n - 1, 1)):
        tile = row // 16 * wide + col // 128
        lane = 16 * (col // 8 % 4) + row % 16
        word = int(words[tile * 256 + lane * 4 + col // 32 % 4]) & 0xFFFFFFFF
        i = col % 8
        bits = [(16 * (i % 2) + 4 * (i // 2) + 3 + b) % 32 for b in range(4)]
        assert sum((word >> bit & 1) << b for b, bit in enumerate(bits)) == int(q[row, col])
        at = m.scales[row // 16, col // group, row % 16]
        assert float(at) == float(scales[row, col // group])
    assert m.nbytes() == m.packed.numel() + m.scales.numel() * 2 + (
        m.scales.numel() if zeros else 0)
    again = W4Matrix(m.packed, m.scales, m.zeros, n, k, group)
    assert torch.equal(again.values()[0], q)


def plain_quantize(w, group, zeros):
    """One group at a time, in Python's 64-bit numbers and fp32 tensors."""

    n, k = w.shape
    groups = -(-k // group)
    q = torch.zeros(n, k, dtype=U8)
    scales = torch.zeros(n, groups, dtype=BF)
    points = torch.zeros(n, groups, dtype=U8)
    for r in range(n):
        for g in range(groups):
            part = [float(v) for v in w[r, g * group:(g + 1) * group]]
            lo, hi = min(part + [0.0]), max(part + [0.0])
            if zeros:
                span = torch.tensor(hi, dtype=torch.float32) - torch.tensor(
                    lo, dtype=torch.float32)
                scale = (span / 15).to(BF)
            else:
                scale = (torch.tensor(max(hi, -lo), dtype=torch.float32) / 7).to(BF)
            scales[r, g] = scale
            s = float(scale)
            zero = 8
            if zeros:
                zero = min(15, max(0, round(-lo / s))) if s else 0
            points[r, g] = zero
            for i, v in enumerate(part):
                q[r, g * group + i] = min(15, max(0, round(v / s) + zero)) if s else zero
    return q, scales, points if zeros else None


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(5, 200, 64), (20, 64, 32), (3, 256, 128)])
def test_quantize(n, k, group, zeros):
    w = normal((n, k), torch.Generator().manual_seed(n * k), 0.02)
    w[0, :group] = 0
    w[1, 3] = 4.0  # an outlier
    w[2] = w[2].abs()  # one sign only
    w[2, :8] = torch.tensor([0.0, -0.0, 0.5, 1.5, 2.5, 3.5, 7.0, 1.0], dtype=BF)
    got = W4Matrix.quantize(w, group=group, zeros=zeros).values()
    want = plain_quantize(w, group, zeros)
    assert torch.equal(got[1], want[1])
    if zeros:
        assert torch.equal(got[2], want[2])
    else:
        assert got[2] is None
    assert torch.equal(got[0], want[0])


def test_quantize_in_pieces(monkeypatch):
    from layer_streaming import w4

    w = normal((100, 72), torch.Generator().manual_seed(3))
    whole = W4Matrix.quantize(w, group=32, zeros=True)
    monkeypatch.setattr(w4, "_PIECE", 2000)
    pieces = W4Matrix.quantize(w, group=32, zeros=True)
    for a, b in zip(whole.values(), pieces.values()):
        assert torch.equal(a, b)
    q, scales, points = whole.values()
    assert torch.equal(W4Matrix.pack(q, scales, zeros=points, group=32).packed, whole.packed)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_no_numbers_has_a_nan_scale(value, zeros):
    w = normal((2, 64), torch.Generator().manual_seed(3))
    w[1, 40] = value
    m = W4Matrix.quantize(w, group=32, zeros=zeros)
    scales = m.values()[1]
    assert bool(scales[1, 1].isnan()) and bool(scales.flatten()[[0, 1, 2]].isfinite().all())


@pytest.mark.parametrize("name,change", [
    ("values", lambda t: t.int()), ("values", lambda t: t[0]), ("values", lambda t: t[:, :12]),
    ("values", lambda t: t + 1), ("values", lambda t: t[:0]), ("values", lambda t: t.tolist()),
    ("scales", lambda t: t.float()), ("scales", lambda t: t[:-1]), ("scales", lambda t: None),
    ("scales", lambda t: t[:, :1]), ("zeros", lambda t: t.int()), ("zeros", lambda t: t[:-1]),
    ("zeros", lambda t: t + 16), ("group", lambda t: 16), ("group", lambda t: 48),
    ("group", lambda t: 64.0), ("group", lambda t: 128)])
def test_pack_refuses(name, change):
    args = dict(values=torch.full((20, 128), 15, dtype=U8),
                scales=torch.ones(20, 2, dtype=BF), zeros=torch.zeros(20, 2, dtype=U8), group=64)
    W4Matrix.pack(**args)
    args[name] = change(args[name])
    with pytest.raises((TypeError, ValueError)):
        W4Matrix.pack(**args)


def test_a_matrix_refuses_parts_of_other_sizes():
    m = W4Matrix.pack(*random_matrix(20, 128, 64, True, 1), group=64)
    good = dict(packed=m.packed, scales=m.scales, zeros=m.zeros, n=20, k=128, group=64)
    W4Matrix(**good)
    for name, value in (("packed", m.packed[:-16]), ("packed", None), ("n", 33), ("n", 0),
                        ("k", 136), ("k", 130), ("group", 32), ("scales", m.scales[:1]),
                        ("zeros", m.scales), ("scales", m.scales.permute(2, 1, 0)),
                        ("packed", torch.zeros(2049, dtype=U8)[1:])):
        with pytest.raises((TypeError, ValueError)):
            W4Matrix(**dict(good, **{name: value}))
    with pytest.raises(AttributeError):
        m.packed = m.packed[:16]
    with pytest.raises(TypeError):
        W4Matrix.quantize(torch.zeros(16, 64))


def linear_args(**changes):
    names = dict(x=16, xs=4096, packed=16, scales=16, zeros=16, m=4, n=100, k=4096, group=128,
                 residual=48, rs=100, y=32, ys=100, workspace=16, workspace_bytes=1 << 40,
                 stream=None)
    assert set(changes) <= set(names)
    names.update(changes)
    return list(names.values())


REFUSED = [
    (1001, dict(x=None)), (1001, dict(packed=None)), (1001, dict(scales=None)),
    (1001, dict(y=None)), (1001, dict(m=0)), (1001, dict(n=0)), (1001, dict(k=0)),
    (1001, dict(xs=4088)), (1001, dict(ys=99)), (1001, dict(y=16)), (1001, dict(rs=-100)),
    (1001, dict(xs=-4096)), (1003, dict(group=16)), (1003, dict(group=256)),
    (1003, dict(group=0)), (1003, dict(m=1 << 30)), (1003, dict(n=1 << 30)),
    (1003, dict(k=1 << 30, xs=1 << 30)), (1002, dict(k=4092)), (1002, dict(x=8)),
    (1002, dict(xs=4100)), (1002, dict(packed=24)), (1002, dict(scales=24)),
    (1002, dict(zeros=24)), (1002, dict(y=33)), (1002, dict(residual=49))]


@pytest.mark.parametrize("code,changes", REFUSED)
def test_linear_entry_point_refuses(code, changes):
    assert _hip.load().cascade_linear_w4_bf16(*linear_args(**changes)) == code


@pytest.mark.parametrize("code,changes", [c for c in REFUSED if not set(c[1]) & {
    "rs", "residual"}] + [(1002, dict(y=34))])
def test_logits_entry_point_refuses(code, changes):
    args = linear_args(**changes)
    assert _hip.load().cascade_linear_w4_f32out_bf16(*args[:9], *args[11:]) == code


@pytest.mark.parametrize("code,changes", [c for c in REFUSED if not set(c[1]) & {
    "rs", "residual", "workspace"}] + [(1001, dict(u_packed=None)), (1001, dict(u_zeros=None)),
                                       (1002, dict(u_scales=20))])
def test_gate_up_entry_point_refuses(code, changes):
    up = {name: changes.pop("u_" + name, 16) for name in ("packed", "scales", "zeros")}
    a = linear_args(**changes)
    args = a[:5] + list(up.values()) + a[5:9] + a[11:13] + [None]
    assert _hip.load().cascade_gate_up_swiglu_w4_bf16(*args) == code


@pytest.mark.parametrize("code,changes", [
    (1004, dict(workspace=None)), (1004, dict(workspace_bytes=4)), (1002, dict(workspace=24))])
def test_a_split_product_refuses(code, changes):
    # 4 rows by 100 x 14336 are split over K
    assert _hip.linear_w4_workspace_bytes(4, 100, 14336) > 4
    args = linear_args(k=14336, xs=14336, **changes)
    assert _hip.load().cascade_linear_w4_bf16(*args) == code
    assert _hip.load().cascade_linear_w4_f32out_bf16(*args[:9], *args[11:]) == code


@pytest.fixture
def launches(monkeypatch):
    calls = []

    def on(name, tensor):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(name)
        return tensor.device

    monkeypatch.setattr(_hip, "_gpu_of", on)
    monkeypatch.setattr(_hip, "_call_on", lambda *args: calls.append(args))
    return calls


def linear_call():
    return _hip.linear_w4, dict(
        x=torch.zeros(3, 64, dtype=BF), out=torch.zeros(3, 40, dtype=BF),
        matrix=W4Matrix.pack(*random_matrix(40, 64, 32, True, 1), group=32),
        residual=torch.zeros(3, 40, dtype=BF), workspace=torch.zeros(64, dtype=U8))


def gate_up_call():
    gate, up = (W4Matrix.pack(*random_matrix(40, 64, 32, True, s), group=32) for s in (1, 2))
    return _hip.gate_up_swiglu_w4, dict(
        x=torch.zeros(3, 64, dtype=BF), out=torch.zeros(3, 40, dtype=BF), gate=gate, up=up)


_wide = lambda t: torch.stack((t, t), -1).flatten(-2)[..., ::2]
_other = lambda n, k, g, z: lambda t: W4Matrix.pack(*random_matrix(n, k, g, z, 1), group=g)
ROWS = [("x", lambda t: t.float()), ("x", lambda t: t[0]), ("x", _wide),
        ("x", lambda t: t[:, :56].contiguous()), ("x", lambda t: None),
        ("out", lambda t: t.double()), ("out", lambda t: t[:-1]), ("out", _wide),
        ("out", lambda t: t[:, :-1]), ("out", lambda t: t[:1].expand_as(t)),
        ("out", lambda t: None)]


@pytest.mark.parametrize("name,change", ROWS + [
    ("matrix", _other(40, 72, 32, True)), ("matrix", _other(48, 64, 32, True)),
    ("matrix", lambda t: t.packed), ("matrix", lambda t: None),
    ("residual", lambda t: t.float()), ("residual", lambda t: t[:-1]), ("residual", _wide),
    ("workspace", lambda t: t.int()), ("workspace", _wide)])
def test_linear_refuses(launches, name, change):
    function, args = linear_call()
    assert function(**args) is args["out"] and len(launches) == 1
    args[name] = change(args[name])
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert len(launches) == 1


@pytest.mark.parametrize("name,change", ROWS + [
    ("gate", _other(40, 72, 32, True)), ("up", _other(40, 72, 32, True)),
    ("up", _other(56, 64, 32, True)), ("up", _other(40, 64, 64, True)),
    ("up", _other(40, 64, 32, False)), ("up", lambda t: None),
    ("gate", lambda t: t.packed), ("out", lambda t: t.float())])
def test_gate_up_refuses(launches, name, change):
    function, args = gate_up_call()
    assert function(**args) is args["out"] and len(launches) == 1
    args[name] = change(args[name])
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert len(launches) == 1


def test_logits_take_no_residual_and_x_is_not_written(launches):
    function, args = linear_call()
    with pytest.raises(ValueError):
        function(**dict(args, out=torch.zeros(3, 40)))
    function(**dict(args, out=torch.zeros(3, 40), residual=None))
    square = W4Matrix.pack(*random_matrix(64, 64, 32, True, 1), group=32)
    with pytest.raises(ValueError):
        function(args["x"], square, args["x"])
    # the residual may be written
    function(**dict(args, residual=args["out"]))
    assert len(launches) == 2


def test_no_rows(launches):
    for call in (linear_call, gate_up_call):
        function, args = call()
        args.update(x=args["x"][:0], out=args["out"][:0])
        if "residual" in args:
            args["residual"] = args["residual"][:0]
        assert function(**args) is args["out"]
    assert not launches


def test_workspaces_of_any_shape():
    size = _hip.linear_w4_workspace_bytes
    for rows in (0, 1, 16, 61, 700):
        for n, k in ((1, 8), (4096, 4096), (4096, 14336), (128256, 4096)):
            assert size(rows, n, k) >= 0 and size(rows, n, k) % 16 == 0
    # whole parts of rows of 16 columns
    assert size(16, 4096, 14336) % (16 * 4096 * 4) == 0 < size(16, 4096, 14336)
    assert size(1, 128256, 4096) == size(700, 4096, 4096) == size(0, 4096, 14336) == 0
