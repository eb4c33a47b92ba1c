"""Refusals of the paged operators' and of sampling's Python wrappers, on the
CPU: the argument is named or typed wrong, and nothing is launched."""

import pytest
import torch

from layer_streaming import _hip
from paged_calls import CALLS, WRONG, ids_of, wrong_call


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(_hip, "_gpu_of", lambda name, t: (
        t.device if isinstance(t, torch.Tensor) else _refuse(name)))
    monkeypatch.setattr(_hip, "_call_on", lambda *args: calls.append(args))
    return calls


def _refuse(name):
    raise TypeError("{} must be a torch.Tensor".format(name))


@pytest.mark.parametrize("which", CALLS)
def test_the_call_itself_is_taken(launches, which):
    function, args = CALLS[which]("cpu")
    function(**args)
    assert len(launches) == 1


@pytest.mark.parametrize("which,names,change", WRONG, ids=ids_of(WRONG))
def test_wrong_arguments_are_refused(launches, which, names, change):
    function, args = wrong_call(which, names, change, "cpu")
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert not launches
