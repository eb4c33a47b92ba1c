"""Settings of a draw without --temperature: the run would be greedy."""

import pytest

from test_cli_sampling_args import parse


@pytest.mark.parametrize("flags", [("--sample-top-k", "40"), ("--sample-top-p", "0.9"),
                                   ("--sample-min-p", "0.05")])
def test_settings_of_a_draw_need_a_temperature(flags, capsys):
    with pytest.raises(SystemExit):
        parse(*flags)
    assert "--temperature" in capsys.readouterr().err
    # greedy by its own flag: nothing is dropped in silence
    assert parse(*flags, "--temperature", "0").temperature == 0
    assert parse(*flags, "--temperature", "0.5").temperature == 0.5


def test_settings_that_are_off_need_none():
    a = parse("--sample-top-k", "0", "--sample-top-p", "1", "--sample-min-p", "0",
              "--sample-seed", "3")
    assert a.temperature == 0
