"""Models in 8 bits, as far as they need no device: the command's options and what is refused."""
from types import SimpleNamespace

import pytest
import torch

import helpers
from tileinfer_b200.cli import COMMANDS, ArgumentError
from tileinfer_b200.config import ApertusConfig
from tileinfer_b200.engine import Engine
from tileinfer_b200.parts import Linear4, Linear8


def test_options():
    for name, rest in (("run", ["m", "1 2"]), ("generate", ["m", "prompts.txt"])):
        values = COMMANDS[name].read(rest)[1]
        assert values["cache"] == values["weights"] == "model"
        assert COMMANDS[name].read(rest + ["--cache", "e4m3"])[1]["cache"] == "e4m3"
        assert COMMANDS[name].read(rest + ["--weights", "e4m3"])[1]["weights"] == "e4m3"
    with pytest.raises(ArgumentError, match="--cache expects model or e4m3"):
        COMMANDS["run"].read(["m", "1", "--cache", "int8"])


def check8(raw=helpers.TINY_B, dtype=torch.bfloat16, kernels="fast", page_size=64, change=None):
    spec = ApertusConfig.from_dict(raw).model_spec()
    if change:
        change(spec)
    Engine._check8(SimpleNamespace(spec=spec, dtype=dtype), kernels, page_size)


def test_what_goes_with_8_bits():
    check8()
    check8(helpers.TINY_C)
    for kw in (dict(dtype=torch.float32), dict(kernels="plain"), dict(page_size=32)):
        with pytest.raises(ValueError, match="bfloat16, the fast kernels and pages of 64"):
            check8(**kw)
    with pytest.raises(ValueError, match="multiple of 16"):
        check8({**helpers.TINY_C, "head_dim": 40})


def test_words_are_checked_before_anything_else():
    for kw in (dict(cache="int8"), dict(weights="fp8")):
        with pytest.raises(ValueError, match="expects model or e4m3"):
            Engine(None, {}, **kw)


def test_matrices_that_do_not_fit():
    rt = SimpleNamespace()
    other = SimpleNamespace(rt=rt, name="up", partials_name="p", out_features=8, in_features=40, weight=torch.zeros(8, 40, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="multiple of 16"):
        Linear8(other)
    other.in_features, other.weight = 64, torch.zeros(8, 64)
    with pytest.raises(ValueError, match="bfloat16"):
        Linear8(other)
    other.weight = None
    for make in (Linear8, lambda o: Linear4(o, 32)):
        with pytest.raises(ValueError):
            make(other)
