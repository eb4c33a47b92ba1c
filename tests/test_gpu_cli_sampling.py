"""Sampled decoding through the run_llama31 CLI: the same tokens from the same
seed with the vocabulary streamed or resident, others from another seed, and
the greedy tokens where the settings leave one."""

import pytest

from test_gpu_cli import run_cli

pytestmark = pytest.mark.gpu


def test_cli_samples_tokens(gpu_device, tmp_path):
    def ids(*flags):
        return run_cli(tmp_path, "--granularity", "layer", "--max-new-tokens", "5",
                       *flags)["generated_ids"]

    hot = ("--temperature", "3.0", "--sample-top-p", "0.99", "--sample-top-k", "5000")
    first = ids("--vocab-mode", "resident", *hot, "--sample-seed", "1")
    # the streamed head draws from the same logits
    assert ids("--vocab-mode", "streamed", *hot, "--sample-seed", "1") == first
    assert ids("--vocab-mode", "resident", *hot, "--sample-seed", "2") != first
    greedy = ids("--vocab-mode", "resident")
    assert ids("--vocab-mode", "resident", "--temperature", "0.9", "--sample-top-k",
               "1") == greedy
    assert ids("--vocab-mode", "resident", "--temperature", "1e-30") == greedy
