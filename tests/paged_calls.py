"""Calls of the paged operators and of sampling as (function, arguments), and
what is wrong with others: each change of one argument has to be refused by
name, before anything is launched."""

import torch

from layer_streaming import _hip

BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def append_call(device):
    z = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.paged_append, dict(
        q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), positions=z(3, dtype=I32),
        k_pages=z(5, 2, 8, 64), v_pages=z(5, 2, 8, 64), page_table=z(4, 3, dtype=I32),
        rows=z(3, dtype=I32), rope=(z(24, 32), z(24, 32)), interleaved=False,
        q_out=z(3, 4, 64), error_flag=z(1, dtype=I32))


def attention_call(device):
    z = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.paged_decode_attention, dict(
        q=z(3, 4, 64), k_pages=z(5, 2, 8, 64), v_pages=z(5, 2, 8, 64),
        page_table=z(4, 3, dtype=I32), lengths=z(4, dtype=I32), out=z(3, 4, 64),
        workspace=z(4096, dtype=torch.uint8), scale=0.125, rows=z(3, dtype=I32),
        max_length=24, error_flag=z(1, dtype=I32))


def sample_call(device):
    z = lambda *shape, dtype=F32: torch.zeros(shape, dtype=dtype, device=device)
    return _hip.sample, dict(
        logits=z(3, 50), uniform=z(3), ids=z(3, dtype=torch.int64),
        workspace=z(4096, dtype=torch.uint8), temperature=z(3), top_k=z(3, dtype=I32),
        top_p=z(3), min_p=z(3), logprobs=z(3))


CALLS = {"append": append_call, "attention": attention_call, "sample": sample_call}

_like = torch.zeros_like


def _wide(t):
    """The same values in every other element of each row."""

    return torch.stack((t, t), -1).flatten(-2)[..., ::2]


def _shared(t):
    """All of the first dimension in one place."""

    return t[:1].expand_as(t)


def _short(t):
    return t[:-1].contiguous()


def _other(t):
    return t.to(torch.float16) if t.dtype != torch.float16 else t.to(BF)


def _heads_first(t):
    return t.transpose(1, 2).contiguous().transpose(1, 2)


POOLS = [
    ("k_pages", _other), ("v_pages", _other), ("v_pages", _short),
    ("k_pages", _wide), ("k_pages", lambda t: t[0]), ("v_pages", _heads_first),
    ("v_pages", lambda t: torch.zeros(5, 2, 16, 64, dtype=BF, device=t.device)[:, :, :8]),
    ("page_table", lambda t: t.long()), ("page_table", lambda t: t[0]),
    ("page_table", _wide), ("page_table", _shared),
    ("page_table", lambda t: t.float()),
    ("rows", lambda t: t.long()), ("rows", _short), ("rows", _wide),
    ("error_flag", lambda t: t.long()), ("error_flag", lambda t: t[:0]),
]

# (call, argument, what becomes of it)
WRONG = [("append", *c) for c in POOLS + [
    ("q", _other), ("q", _short), ("q", _wide), ("q", lambda t: t[..., :32].contiguous()),
    ("q", lambda t: t[0]), ("q", lambda t: None), ("q", lambda t: t.tolist()),
    ("k", _other), ("k", _short), ("k", _wide), ("k", lambda t: t[:, :1].contiguous()),
    ("k", lambda t: t[0]), ("k", lambda t: None), ("v", _other), ("v", _short),
    ("v", _wide), ("v", lambda t: None),
    ("positions", lambda t: t.long()), ("positions", _short), ("positions", _wide),
    ("positions", lambda t: t[:, None]), ("positions", lambda t: None),
    ("rope", lambda t: (t[0], t[1][:-1])), ("rope", lambda t: (_wide(t[0]), t[1])),
    ("rope", lambda t: (t[0], t[1].float())), ("rope", lambda t: (t[0][0], t[1][0])),
    ("rope", lambda t: t[0]), ("q_out", _other), ("q_out", _short), ("q_out", _wide),
    ("q_out", _shared), ("q_out", lambda t: t[:, :1].expand_as(t)),
    ("q_out", lambda t: torch.as_strided(
        torch.zeros(1000, dtype=BF, device=t.device), t.shape, (224, 64, 1))),
    # without rows, a token a table row
    ("page_table,rows", lambda t: (t[0][:2].contiguous(), None)),
]] + [("attention", *c) for c in POOLS + [
    ("q", _other), ("q", _short), ("q", _wide), ("q", lambda t: t[..., :32].contiguous()),
    ("q", lambda t: t[0]), ("q", lambda t: None),
    ("out", _other), ("out", _short), ("out", _wide), ("out", _shared),
    ("out", lambda t: t[:, :1].expand_as(t)), ("out", lambda t: None),
    ("lengths", lambda t: t.long()), ("lengths", _short), ("lengths", _wide),
    ("lengths", lambda t: None), ("workspace", lambda t: t.view(torch.int8)),
    ("workspace", lambda t: t.view(64, 64)), ("workspace", _wide),
    ("workspace", lambda t: None), ("max_length", lambda t: 0), ("max_length", lambda t: -1),
    ("max_length", lambda t: 25),
    ("page_table,lengths,rows", lambda t: (t[0][:2].contiguous(), t[1][:2].contiguous(),
                                           None)),
]] + [("sample", *c) for c in [
    ("logits", lambda t: t.double()), ("logits", lambda t: t[0]), ("logits", _wide),
    ("logits", _shared), ("logits", lambda t: None), ("uniform", lambda t: t.double()),
    ("uniform", _short), ("uniform", _wide), ("uniform", lambda t: 0.5),
    ("ids", lambda t: t.int()), ("ids", _short), ("ids", _wide), ("ids", lambda t: None),
    ("workspace", lambda t: t.view(torch.int8)), ("workspace", _wide),
    ("logprobs", lambda t: t.double()), ("logprobs", _short), ("logprobs", _wide),
    ("temperature", lambda t: t.double()), ("temperature", _short),
    ("temperature", lambda t: t[0]), ("top_k", lambda t: t.long()), ("top_k", _wide),
    ("top_p", _short), ("top_p", lambda t: t.to(BF)), ("min_p", _wide),
    ("min_p", lambda t: t[:, None]),
]]


def wrong_call(which, names, change, device):
    function, args = CALLS[which](device)
    names = names.split(",")
    if len(names) == 1:
        args[names[0]] = change(args[names[0]])
    else:
        args.update(zip(names, change([args[n] for n in names])))
    return function, args


def ids_of(cases):
    seen = {}
    out = []
    for which, names, _ in cases:
        key = "{}-{}".format(which, names)
        seen[key] = seen.get(key, 0) + 1
        out.append("{}-{}".format(key, seen[key]))
    return out
