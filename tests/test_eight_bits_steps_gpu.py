"""Engines with an 8-bit cache, step by step: what steps of other sizes leave standing."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu

HEAD128 = {**helpers.TINY_B, "hidden_size": 192, "num_attention_heads": 32, "num_key_value_heads": 4, "head_dim": 128, "intermediate_size": 272, "vocab_size": 333,
           "num_hidden_layers": 2, "max_position_embeddings": 16384}


@pytest.fixture(scope="module")
def ti():
    import tileinfer_b200
    return tileinfer_b200


def test_longer_prompts_leave_captured_steps_standing(ti):
    """Chunks of one size over ever more positions: the pages that are widened for them grow, no scratch buffer does, and none of it is held afterwards."""
    from tileinfer_b200.config import ApertusConfig
    from tileinfer_b200.kernels import ops
    engine = ti.Engine.random(ApertusConfig.from_dict(HEAD128), seed=1, max_tokens=16384, max_seqs=2, max_context=16384, max_step_tokens=512, cache="e4m3")
    short, long = engine.new_sequence(), engine.new_sequence()
    engine.step([(short, list(range(1, 301)))])
    engine.step([(long, [1] * 512)])
    engine.step([(short, [7])])
    assert engine.graph_ready(1)
    before, held = engine.rt.generation, torch.cuda.memory_allocated()
    needs = set()
    while engine.sequence_length(long) < 13 * 1024:
        engine.step([(long, [(i * 7 + 3) % 333 for i in range(512)])])
        needs.add(ops.attention8_workspace(1, 512, 32, 4, 128, engine.sequence_length(long)))
        assert engine.graph_ready(1) and engine.rt.generation == before
    assert max(needs) > 24 << 20 and len(needs) > 20
    assert torch.cuda.memory_allocated() - held < 1 << 20
    launches = engine.decode_launches(1)
    engine.step([(short, [9])])
    assert engine.graph_ready(1) and engine.decode_launches(1) == launches
    engine.check_health()
