"""Sampling flags of tools/run_llama31.py on the CPU: greedy by default, and
combinations that are refused."""

import pytest


def parse(*argv):
    from tools import run_llama31

    return run_llama31.parse_args(["--random-init", *argv])


def test_defaults_are_greedy():
    a = parse()
    assert (a.temperature, a.sample_top_k, a.sample_top_p, a.sample_min_p) == (0, 0, 1, 0)
    b = parse("--temperature", "0.7", "--sample-top-k", "40", "--sample-top-p", "0.9",
              "--sample-min-p", "0.05", "--sample-seed", "11")
    assert (b.temperature, b.sample_top_k, b.sample_top_p, b.sample_min_p,
            b.sample_seed) == (0.7, 40, 0.9, 0.05, 11)


@pytest.mark.parametrize("flags", [
    ("--temperature", "-1"), ("--temperature", "nan"), ("--sample-top-k", "-1"),
    ("--sample-top-p", "-0.1"), ("--sample-min-p", "-0.1"),
    ("--decode-graph", "--vocab-mode", "resident", "--temperature", "0.5")])
def test_refused(flags):
    with pytest.raises(SystemExit):
        parse(*flags)
