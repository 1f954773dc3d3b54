"""What goes with a cache in 8 bits and what with matrices in 8 bits: each is asked about its own sizes alone, before anything is loaded."""
from types import SimpleNamespace

import pytest
import torch

import helpers
from tileinfer_b200.config import ApertusConfig
from tileinfer_b200.engine import Engine


def check8(cache, weights, raw=helpers.TINY_B, dtype=torch.bfloat16, kernels="fast", page_size=64):
    spec = ApertusConfig.from_dict(raw).model_spec()
    Engine._check8(SimpleNamespace(spec=spec, dtype=dtype), kernels, page_size, cache, weights)


def test_matrices_alone_go_with_any_pages_and_heads():
    check8(False, True, page_size=32)
    check8(False, True, {**helpers.TINY_B, "head_dim": 40, "num_attention_heads": 6})
    check8(False, True, {**helpers.TINY_B, "head_dim": 272, "num_attention_heads": 1, "num_key_value_heads": 1})
    for kw in (dict(page_size=32), dict(raw={**helpers.TINY_B, "head_dim": 40}), dict(raw={**helpers.TINY_B, "head_dim": 272})):
        with pytest.raises(ValueError, match="pages of 64|multiple of 16"):
            check8(True, False, **kw)


def test_the_cache_alone_goes_with_any_matrices():
    raw = {**helpers.TINY_B, "hidden_size": 100, "intermediate_size": 321}
    check8(True, False, raw)
    for change in (dict(hidden_size=100), dict(intermediate_size=321), dict(head_dim=40, num_attention_heads=3)):
        with pytest.raises(ValueError, match="multiple of 16 inputs, not (100|321|120)"):
            check8(False, True, {**helpers.TINY_B, **change})


@pytest.mark.parametrize("cache,weights", [(True, False), (False, True), (True, True)])
def test_both_want_bfloat16_and_the_fast_kernels(cache, weights):
    check8(cache, weights)
    for kw in (dict(dtype=torch.float32), dict(kernels="plain")):
        with pytest.raises(ValueError, match="bfloat16.* the fast kernels"):
            check8(cache, weights, **kw)


@pytest.mark.gpu
def test_matrices_in_8_bits_with_small_pages_and_odd_heads():
    """The same tokens whatever the pages' size, and a step's logits near the bfloat16 model's (a product's factors are off by 2.6 % each on average)."""
    import tileinfer_b200 as ti
    raw = {**helpers.TINY_B, "head_dim": 40}
    config = ApertusConfig.from_dict(raw)
    make = lambda **kw: ti.Engine.random(config, seed=1, max_tokens=1024, max_seqs=2, max_context=256, **kw)  # noqa: E731
    prompts = helpers.random_prompts(config.vocab_size, [3, 70], 4)
    engines = [make(weights="e4m3", page_size=page) for page in (32, 64)]
    outs = [ti.generate(e, prompts, max_new_tokens=20, stop_ids=[]) for e in engines]
    assert outs[0] == outs[1]
    plain = make()
    logits = [e.step([(e.new_sequence(), prompts[1])]).double() for e in (engines[0], plain)]
    assert 0 < float((logits[0] - logits[1]).norm() / logits[1].norm()) < 0.2
    for e in engines:
        e.check_health()
