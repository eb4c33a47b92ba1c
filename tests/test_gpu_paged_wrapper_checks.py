"""The wrappers' two ways through their checks, with tensors on the GPU: what
the short expression takes, the checks one by one take with the same
arguments, and neither takes a wrong one.  Nothing is launched."""

import pytest
import torch

from layer_streaming import _hip
from paged_calls import CALLS, WRONG, ids_of, wrong_call

pytestmark = pytest.mark.gpu

TENSORS = [(which, name) for which in CALLS
           for name, value in CALLS[which]("cpu")[1].items()
           if isinstance(value, (torch.Tensor, tuple))]


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(_hip, "_call_on", lambda *args: calls.append(args))
    return calls


@pytest.mark.parametrize("which,names,change", WRONG, ids=ids_of(WRONG))
def test_wrong_arguments_are_refused(gpu_device, launches, which, names, change):
    function, args = wrong_call(which, names, change, gpu_device)
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert not launches


@pytest.mark.parametrize("which,name", TENSORS)
def test_tensors_on_the_host_are_refused(gpu_device, launches, which, name):
    function, args = CALLS[which](gpu_device)
    value = args[name]
    args[name] = (value[0], value[1].cpu()) if isinstance(value, tuple) else value.cpu()
    with pytest.raises((TypeError, ValueError)):
        function(**args)
    assert not launches


def forms(which, device):
    """Calls of the ordinary form: all arguments, the optional ones left out,
    single heads, tokens and table rows."""

    function, args = CALLS[which](device)
    yield function, args
    few = dict(args, error_flag=None, rows=None)
    if which == "append":
        yield function, dict(few, rope=None)
        yield function, dict(few, q=None, q_out=None)
        fused = torch.zeros(3, 8, 64, dtype=torch.bfloat16, device=device)
        yield function, dict(few, q=fused[:, :4], k=fused[:, 4:6], v=fused[:, 6:])
        one = dict(few, q=fused[:1, :1], k=fused[:1, 1:2], v=fused[:1, 2:3],
                   q_out=torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=device),
                   positions=args["positions"][:1],
                   k_pages=args["k_pages"][:, :1], v_pages=args["v_pages"][:, :1])
        yield function, one
        yield function, dict(one, page_table=args["page_table"][:1])
    else:
        yield function, few
        fused = torch.zeros(3, 8, 64, dtype=torch.bfloat16, device=device)
        yield function, dict(few, q=fused[:, 2:6])
        one = dict(few, q=fused[:1, :1], out=args["out"][:1, :1].contiguous(),
                   k_pages=args["k_pages"][:, :1], v_pages=args["v_pages"][:, :1])
        yield function, one
        yield function, dict(one, page_table=args["page_table"][:1],
                             lengths=args["lengths"][:1])


@pytest.mark.parametrize("which", ["append", "attention"])
def test_both_ways_give_the_same_arguments(gpu_device, launches, monkeypatch, which):
    check = "_check_append" if which == "append" else "_check_attention"
    one_by_one, checked = getattr(_hip, check), []
    monkeypatch.setattr(_hip, check, lambda *a: checked.append(a) or one_by_one(*a))
    for function, args in forms(which, gpu_device):
        function(**args)
        assert not checked, "taken for unordinary"
        with monkeypatch.context() as m:
            m.setattr(_hip, "_I32", None)  # no type is the ordinary one
            function(**args)
        assert len(checked) == 1 and len(launches) == 2
        # (but for the output's strides of dimensions of one, which say nothing)
        size = (args["q_out"] if which == "append" else args["out"])
        size = None if size is None else size.shape[:2]
        at = 28 if which == "append" else 24
        loose = [at + i for i in (0, 1) if size is not None and size[i] == 1]
        pairs = [pair for i, pair in enumerate(zip(*launches)) if i not in loose]
        assert len(launches[0]) == len(launches[1]) and all(a == b for a, b in pairs)
        checked.clear()
        launches.clear()
