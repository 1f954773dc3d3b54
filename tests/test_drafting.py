"""Drafted generation, as far as it needs no device: the command's option and what a draft refuses."""
from types import SimpleNamespace

import pytest

from tileinfer_b200.cli import COMMANDS, ArgumentError, drafted, load_draft
from tileinfer_b200.engine import Draft, generate
from tileinfer_b200.engine.drafting import quantized


def test_option():
    for name, rest in (("run", ["m", "1 2"]), ("generate", ["m", "prompts.txt"])):
        command = COMMANDS[name]
        assert command.read(rest)[1]["draft"] == 0
        values = command.read(rest + ["--draft", "4"])[1]
        assert values["draft"] == 4
    with pytest.raises(ArgumentError, match="--draft expects an integer"):
        COMMANDS["run"].read(["m", "1", "--draft", "few"])
    assert load_draft(None, {"draft": 0}) is None
    assert drafted(None) == "" and drafted(SimpleNamespace(stood=3, drafted=8)) == "; 3 of 8 drafted tokens stood"


def engine(rolls_back=True, windowed=()):
    return SimpleNamespace(cache=SimpleNamespace(groups=[SimpleNamespace(rolls_back=rolls_back)], windowed_groups=list(windowed)))


def test_a_draft_refuses():
    with pytest.raises(ValueError, match="at least one token"):
        Draft(engine(), 0)
    for e in (engine(rolls_back=False), engine(windowed=[0])):
        with pytest.raises(ValueError, match="cut back"):
            Draft(e, 4)
    with pytest.raises(ValueError, match="another engine"):
        generate(SimpleNamespace(), [[1]], 4, draft=SimpleNamespace(engine=None))


def test_only_known_layers_become_four_bits():
    layer = SimpleNamespace(mixer=SimpleNamespace(kind="attention"), feed_forward=SimpleNamespace(kind="routed"))
    with pytest.raises(ValueError, match="not of attention and routed"):
        quantized(SimpleNamespace(spec=SimpleNamespace(layers=[layer])))
