"""Log-probabilities of drawn tokens, however unlikely, against 64 bits."""

import math

import pytest
import torch

from test_gpu_sample import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [40, 20000])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=30), dict(top_k=300),
                                      dict(temperature=0.7)], ids=str)
def test_log_probability_of_unlikely_tokens(gpu_device, vocab, settings):
    # uniform 0 takes the first token with a weight: token 0, at 2^-10 to 2^-44
    # of the likeliest, which is the last
    temperature = settings.get("temperature", 1.0)
    below = torch.tensor([10.0, 20.0, 30.0, 38.0, 41.0, 43.0, 43.7, 44.2]) * math.log(2.0)
    logits = torch.full((8, vocab), -math.inf)
    logits[:, 0] = -below * temperature
    logits[:, 1] = -3.0
    logits[:, vocab - 1] = 0.0
    ids, logprobs = draw(logits, torch.zeros(8), gpu_device, **settings)
    assert ids.tolist() == [0] * 8
    x = logits.double() / temperature
    exact = x[:, 0] - torch.logsumexp(x, 1)
    # the sum of three weights that are multiples of 2^-44 of the largest,
    # half a step each; a few roundings in 64 bits; one rounding to fp32
    tol = 2.0 ** -24 * exact.abs() + 3 * 2.0 ** -45 + 2.0 ** -45
    assert bool(((logprobs.double() - exact).abs() <= tol).all()), logprobs - exact
