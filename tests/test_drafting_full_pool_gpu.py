"""Generation with a draft where the plan fills the pool to its last page and the sequences end at different times."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
PAGE = 64


@pytest.fixture(scope="module")
def ti():
    import tileinfer_b200
    return tileinfer_b200


def make(ti, lengths, budget, dtype="float32"):
    from tileinfer_b200.config import ApertusConfig
    cfg = ApertusConfig.from_dict(helpers.TINY_B)
    pool = sum(-(-(n + budget) // PAGE) * PAGE for n in lengths)
    engine = ti.Engine.random(cfg, seed=1, dtype=dtype, max_tokens=pool, max_seqs=len(lengths), max_context=512)
    return engine, helpers.random_prompts(cfg.vocab_size, lengths, 3)


class Uneven:
    """A draft whose proposals are spoiled for some slots, so that progress is unequal whatever the weights say."""

    def __init__(self, draft, spoiled):
        self.inner, self.spoiled, self.propose_inner = draft, spoiled, draft.propose
        draft.propose = self.propose

    def propose(self, slots, last, k, sampling, seeds, counters, counts=None):
        drafts, q = self.propose_inner(slots, last, k, sampling, seeds, counters, counts)
        for row, slot in enumerate(slots):
            if slot in self.spoiled:
                drafts[row] = (drafts[row] + 1) % self.inner.engine.vocab_size
        return drafts, q


@pytest.mark.parametrize("lengths,budget", [((44, 44), 20), ((120, 120), 8), ((44, 108, 30, 51), 20)])
@pytest.mark.parametrize("tokens", [2, 4])
def test_the_models_tokens_on_a_full_pool(ti, lengths, budget, tokens):
    engine, prompts = make(ti, lengths, budget)
    want = ti.generate(engine, prompts, max_new_tokens=budget, stop_ids=[])
    draft = ti.Draft(engine, tokens=tokens, group=32)
    draft.twin = engine.twin(engine.model)                   # a perfect draft, spoiled for every other sequence
    Uneven(draft, {0, 2})
    assert ti.generate(engine, prompts, max_new_tokens=budget, stop_ids=[], draft=draft) == want
    assert 0 < draft.stood < draft.drafted and engine.cache.lengths == {}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampled_on_a_full_pool(ti, dtype):
    lengths, budget = (44, 108, 30, 51), 20
    engine, prompts = make(ti, lengths, budget, dtype)
    draft = ti.Draft(engine, tokens=4, group=32)
    sampling = ti.SamplingParams(temperature=0.9, top_k=30)
    out = ti.generate(engine, prompts, max_new_tokens=budget, sampling=sampling, stop_ids=[], draft=draft, seed=5)
    assert [len(o) for o in out] == [budget] * 4
    assert out == ti.generate(engine, prompts, max_new_tokens=budget, sampling=sampling, stop_ids=[], draft=draft, seed=5)
    if dtype == "float32":
        slot = engine.new_sequence()                         # every token is one of the thirty that the model draws from at its place
        for prompt, tokens in zip(prompts, out):
            engine.truncate(slot, 0)
            logits = engine.step([(slot, prompt + tokens)], [list(range(len(prompt) - 1, len(prompt) + len(tokens) - 1))])
            best = logits.topk(30).indices
            assert all(t in best[i].tolist() for i, t in enumerate(tokens))
        engine.free_sequence(slot)
