"""Command line: options that would do nothing are refused before a model is loaded."""
import pytest

from wayruntime_b200 import cli


@pytest.mark.parametrize("option, value", [("--temperature", "0.5"), ("--top-k", "5"), ("--top-p", "0.9"), ("--seed", "3")])
def test_sampling_options_beside_beams(capsys, monkeypatch, option, value):
    monkeypatch.setattr(cli, "generate", lambda a: pytest.fail("not refused"))
    with pytest.raises(SystemExit) as e:
        cli.main(["generate", "--model", "x", "--prompt", "1", "--beams", "2", option, value])
    said = capsys.readouterr().err
    assert e.value.code == 2 and "--beams" in said and option in said


def test_beams_and_sampling_by_themselves(monkeypatch):
    monkeypatch.setattr(cli, "generate", lambda a: 0)
    assert cli.main(["generate", "--model", "x", "--prompt", "1", "--beams", "2", "--length-penalty", "0.5", "--stop", "3"]) == 0
    assert cli.main(["generate", "--model", "x", "--prompt", "1", "--temperature", "0.5", "--top-k", "5", "--top-p", "0.9", "--seed", "3"]) == 0
