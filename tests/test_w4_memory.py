"""The memory that a 4-bit matrix hands to a launch, on the CPU."""

import copy
import io
import pickle

import pytest
import torch

from layer_streaming import W4Matrix, _hip
from w4_cases import random_matrix

BF, U8 = torch.bfloat16, torch.uint8
PARTS = ("packed", "scales", "zeros")


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(_hip, "_gpu_of", lambda name, tensor: tensor.device)
    monkeypatch.setattr(_hip, "_call_on", lambda *args: calls.append(args))
    return calls


def made(seed=1):
    return W4Matrix.pack(*random_matrix(40, 64, 32, True, seed), group=32)


def calls_of(matrix):
    x, out = torch.zeros(3, 64, dtype=BF), torch.zeros(3, 40, dtype=BF)
    return ((_hip.linear_w4, (x, matrix, out)), (_hip.gate_up_swiglu_w4, (x, made(2), matrix, out)),
            (_hip.gate_up_swiglu_w4, (x, matrix, made(2), out)))


def addresses(matrix):
    return tuple(getattr(matrix, name).data_ptr() for name in PARTS)


@pytest.mark.parametrize("name", PARTS)
def test_other_memory_for_a_part_changes_nothing(launches, name):
    # the tensor that was given and the one that is handed out
    whole = made()
    given = {part: getattr(whole, part).clone() for part in PARTS}
    m = W4Matrix(n=40, k=64, group=32, **given)
    at, values = addresses(m), [v.clone() for v in m.values()]
    for tensor in (given[name], getattr(m, name)):
        tensor.set_(torch.zeros(1, dtype=tensor.dtype))
        assert addresses(m) == at == m.launch[1:4]
        for a, b in zip(m.values(), values):
            assert torch.equal(a, b)
    getattr(m, name).data = torch.zeros(1, dtype=given[name].dtype)
    assert addresses(m) == at == m.launch[1:4]
    for function, args in calls_of(m):
        function(*args)
    assert all(at[0] in call for call in launches) and len(launches) == 3


@pytest.mark.parametrize("name", PARTS)
def test_released_memory_is_refused(launches, name):
    m = made()
    storage = getattr(m, name).untyped_storage()
    size = storage.nbytes()
    for less in (0, size - 1):
        storage.resize_(less)
        for function, args in calls_of(m):
            with pytest.raises(ValueError, match="released"):
                function(*args)
        assert not launches
    # and taken where it is back, wherever that is
    storage.resize_(size)
    assert m.launch[1:4] == addresses(m)
    for function, args in calls_of(m):
        function(*args)
    assert len(launches) == 3


def test_parts_of_one_buffer(launches):
    # at their places in a larger storage
    whole = made()
    sizes = [getattr(whole, name).numel() * getattr(whole, name).element_size()
             for name in PARTS]
    starts = [16, 16 + sizes[0] + 32, 16 + sizes[0] + 32 + -(-sizes[1] // 16) * 16]
    buffer = torch.zeros(starts[2] + sizes[2], dtype=U8)
    parts = {}
    for name, start, size in zip(PARTS, starts, sizes):
        part = getattr(whole, name)
        parts[name] = buffer[start:start + size].view(part.dtype).view(part.shape)
        parts[name].copy_(part)
    m = W4Matrix(n=40, k=64, group=32, **parts)
    assert [a - buffer.data_ptr() for a in m.launch[1:4]] == starts
    for a, b in zip(m.values(), whole.values()):
        assert torch.equal(a, b)
    buffer.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="released"):
        m.launch


def pickled(m):
    return pickle.load(io.BytesIO(pickle.dumps(m)))


@pytest.mark.parametrize("twin", [copy.copy, copy.deepcopy, pickled])
def test_a_copy_has_the_addresses_of_its_own_parts(twin):
    m = made()
    other = twin(m)
    assert other.launch[1:4] == addresses(other) and other.launch[4:] == (40, 64, 32)
    for a, b in zip(other.values(), m.values()):
        assert torch.equal(a, b)
    if twin is not copy.copy:
        assert not set(addresses(other)) & set(addresses(m))
        m.packed.untyped_storage().resize_(0)
        other.launch
        other.packed.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match="released"):
            other.launch
