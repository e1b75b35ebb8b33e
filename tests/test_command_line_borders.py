"""Options of the command line that mean nothing together are refused before anything is loaded."""
import pytest

from mllm_b200 import __main__ as cli


@pytest.mark.parametrize("options, what", [(["--pages", "40"], "--page"), (["--temperature", "0.8"], "--draft")])
def test_options_without_the_one_they_belong_to(options, what, capsys):
    with pytest.raises(SystemExit) as e:
        cli.main(["generate", "--model", "/nowhere", "--tokens", "1,2", "--max-new", "3"] + options)
    assert e.value.code == 2 and what in capsys.readouterr().err
