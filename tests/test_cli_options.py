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


def test_a_search_that_finds_nothing(capsys, monkeypatch):
    """Logits that are not numbers have no continuations."""
    import json
    from types import SimpleNamespace
    from wayruntime_b200 import binding, engine, models
    thing = SimpleNamespace(close=lambda: None)
    monkeypatch.setattr(binding, "Context", lambda *a, **kw: thing)
    monkeypatch.setattr(models, "load", lambda *a: thing)
    monkeypatch.setattr(engine, "Engine", lambda m: SimpleNamespace(beam_search=lambda *a: []))
    assert cli.main(["generate", "--model", "x", "--prompt", "1,2", "--beams", "2"]) == 0
    assert json.loads(capsys.readouterr().out) == {"prompt": [1, 2], "output": [], "score": None, "beams": []}
