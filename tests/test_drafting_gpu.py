"""Generation with a draft of the model in 4 bits: the tokens that it leaves, the cache that it leaves, and what it refuses."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ti():
    import tileinfer_b200
    return tileinfer_b200


def make(ti, raw, dtype, seed=1, **kw):
    from tileinfer_b200.config import ApertusConfig
    cfg = ApertusConfig.from_dict(raw)
    return cfg, ti.Engine.random(cfg, seed=seed, dtype=dtype, **{**dict(max_tokens=4096, max_seqs=8, max_context=512), **kw})


@pytest.mark.parametrize("raw", [helpers.TINY_A, helpers.TINY_B])
@pytest.mark.parametrize("tokens", [1, 3, 6])
def test_greedy_tokens_are_the_models_own(ti, raw, tokens):
    """32-bit: a token's logits do not depend on how a step is cut, so drafted and plain generation agree token for token."""
    cfg, engine = make(ti, raw, "float32")
    prompts = helpers.random_prompts(cfg.vocab_size, [1, 4, 17, 33, 70], 3)
    want = ti.generate(engine, prompts, max_new_tokens=20, stop_ids=[])
    draft = ti.Draft(engine, tokens=tokens, group=32)
    seen = []
    got = ti.generate(engine, prompts, max_new_tokens=20, stop_ids=[], draft=draft, on_token=lambda r, t: seen.append((r, t)))
    assert got == want
    for r, tokens_of in enumerate(got):
        assert [t for q, t in seen if q == r] == tokens_of
    assert draft.drafted > 0 and 0 <= draft.stood <= draft.drafted
    assert engine.cache.lengths == {} and ti.generate(engine, prompts, max_new_tokens=20, stop_ids=[]) == want     # every page and slot is back


def test_stop_tokens_and_budgets(ti):
    cfg, engine = make(ti, helpers.TINY_B, "float32")
    prompts = helpers.random_prompts(cfg.vocab_size, [5, 9, 30], 7)
    plain = ti.generate(engine, prompts, max_new_tokens=16, stop_ids=[])
    stop = [plain[1][5]]
    draft = ti.Draft(engine, tokens=4, group=32)
    for budget in (0, 1, 2, 5, 16):
        assert ti.generate(engine, prompts, max_new_tokens=budget, stop_ids=stop, draft=draft) == \
            ti.generate(engine, prompts, max_new_tokens=budget, stop_ids=stop)


def test_a_perfect_draft_stands(ti):
    """A draft of the model itself (its own matrices): every drafted token stands, in 32-bit exactly."""
    cfg, engine = make(ti, helpers.TINY_B, "float32")
    draft = ti.Draft(engine, tokens=4, group=32)
    draft.twin = engine.twin(engine.model)
    prompts = helpers.random_prompts(cfg.vocab_size, [3, 40], 5)
    assert ti.generate(engine, prompts, max_new_tokens=21, stop_ids=[], draft=draft) == ti.generate(engine, prompts, max_new_tokens=21, stop_ids=[])
    assert draft.stood == draft.drafted == 4 * 4 * 2
    # Sampled: what a draft draws from the model's own probabilities stands, too.
    draft.drafted = draft.stood = 0
    sampling = ti.SamplingParams(temperature=0.9, top_k=30, top_p=0.95)
    out = ti.generate(engine, prompts, max_new_tokens=21, sampling=sampling, stop_ids=[], draft=draft, seed=5)
    assert [len(o) for o in out] == [21, 21] and draft.stood == draft.drafted


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampled_tokens_come_from_the_model(ti, dtype):
    """Every token has positive probability under the model's settings at its place, and the same seed gives the same tokens."""
    cfg, engine = make(ti, helpers.TINY_A, dtype)
    draft = ti.Draft(engine, tokens=3, group=32, zeros=True)
    prompts = helpers.random_prompts(cfg.vocab_size, [2, 11, 25], 11)
    sampling = ti.SamplingParams(temperature=0.8, top_k=12)
    out = ti.generate(engine, prompts, max_new_tokens=13, sampling=sampling, stop_ids=[], draft=draft, seed=3)
    assert out == ti.generate(engine, prompts, max_new_tokens=13, sampling=sampling, stop_ids=[], draft=draft, seed=3)
    assert out != ti.generate(engine, prompts, max_new_tokens=13, sampling=sampling, stop_ids=[], draft=draft, seed=4)
    if dtype == "float32":
        slot = engine.new_sequence()
        for prompt, tokens in zip(prompts, out):
            engine.truncate(slot, 0)
            logits = engine.step([(slot, prompt + tokens)], [list(range(len(prompt) - 1, len(prompt) + len(tokens) - 1))])
            best = logits.topk(12).indices
            assert all(t in best[i].tolist() for i, t in enumerate(tokens))
        engine.free_sequence(slot)


def test_first_tokens_follow_the_model(ti):
    """The first two tokens of many sampled runs: the second is drafted and tested. Its frequencies, given the most frequent first token, within five
    standard deviations of the model's probabilities."""
    cfg, engine = make(ti, helpers.TINY_A, "float32", max_seqs=64, max_tokens=64 * 64)
    draft = ti.Draft(engine, tokens=2, group=32)
    sampling = ti.SamplingParams(temperature=0.7, top_k=4)
    prompt = helpers.random_prompts(cfg.vocab_size, [9], 2)[0]
    outs = ti.generate(engine, [prompt] * 2048, max_new_tokens=3, sampling=sampling, stop_ids=[], draft=draft, seed=9)
    firsts = [o[0] for o in outs]
    top = max(set(firsts), key=firsts.count)
    seconds = [o[1] for o in outs if o[0] == top]
    slot = engine.new_sequence()
    logits = engine.step([(slot, prompt + [top])])
    engine.free_sequence(slot)
    z, ids = (logits[0].double() / 0.7).topk(4)
    p = torch.softmax(z, 0)
    for i, pi in zip(ids.tolist(), p.tolist()):
        assert abs(seconds.count(i) / len(seconds) - pi) <= 5 * (pi * (1 - pi) / len(seconds)) ** 0.5
    assert set(seconds) <= set(ids.tolist())


def test_a_few_tokens_step_in_bfloat16(ti):
    """Logits of a step of several tokens a sequence, attention shared out by the caches' lengths or by the tokens: the same up to rounding."""
    cfg, engine = make(ti, helpers.TINY_B, "bfloat16", max_tokens=8192, max_context=1024)
    from tileinfer_b200.kernels import library
    prompts = helpers.random_prompts(cfg.vocab_size, [300, 5, 64, 611], 13)
    runs = helpers.random_prompts(cfg.vocab_size, [5, 5, 2, 4], 14)
    slots = [engine.new_sequence() for _ in prompts]
    engine.step(list(zip(slots, prompts)))
    want = [list(range(len(r))) for r in runs]
    by_tokens = engine.step(list(zip(slots, runs)), want)
    for s, p in zip(slots, prompts):
        engine.truncate(s, len(p))
    before = library.call_counts.get("ti_attention_few", 0)
    by_length = engine.step(list(zip(slots, runs)), want, few=True)
    assert library.call_counts["ti_attention_few"] == before + cfg.num_hidden_layers
    # Both round P and O to bfloat16 in every layer; the model's logits differ by a few of its roundings.
    assert float((by_length - by_tokens).abs().max()) <= 8 * 2.0 ** -8 * float(by_tokens.abs().max())
    for s in slots:
        engine.free_sequence(s)


def test_a_draft_in_bfloat16_of_several_sequences(ti):
    """More than eight sequences (the products' other kernel) through captured steps; the greedy tokens are the model's choices up to near-ties."""
    raw = {**helpers.TINY_B, "hidden_size": 512, "num_attention_heads": 8, "num_key_value_heads": 4, "head_dim": 64, "intermediate_size": 2048, "vocab_size": 4096}
    cfg, engine = make(ti, raw, "bfloat16", max_seqs=12, max_tokens=12 * 256, max_context=256)
    prompts = helpers.random_prompts(cfg.vocab_size, [3, 9, 20, 40, 5, 6, 7, 8, 9, 10, 11, 64], 17)
    draft = ti.Draft(engine, tokens=4)
    outs = ti.generate(engine, prompts, max_new_tokens=12, stop_ids=[], draft=draft)
    engine.check_health()
    slot = engine.new_sequence()
    for prompt, tokens in zip(prompts, outs):
        engine.truncate(slot, 0)
        logits = engine.step([(slot, prompt + tokens)], [list(range(len(prompt) - 1, len(prompt) + len(tokens) - 1))])
        bound = 8 * 2.0 ** -8 * float(logits.abs().max())
        gaps = logits.max(1).values - logits.gather(1, torch.tensor(tokens, device="cuda")[:, None])[:, 0]
        assert float(gaps.max()) <= bound
    engine.free_sequence(slot)


def test_refusals(ti):
    from tileinfer_b200.config import config_from_dict
    cfg, engine = make(ti, helpers.TINY_A, "float32")
    _, other = make(ti, helpers.TINY_A, "float32")
    with pytest.raises(ValueError, match="at least one token"):
        ti.Draft(engine, tokens=0)
    with pytest.raises(ValueError, match="another engine"):
        ti.generate(other, [[1, 2]], max_new_tokens=2, draft=ti.Draft(engine, group=32))
    odd = {**helpers.TINY_A, "hidden_size": 80}
    _, engine = make(ti, odd, "float32")
    with pytest.raises(ValueError, match="groups"):
        ti.Draft(engine)
    import zudepel_cases
    cfg = config_from_dict(zudepel_cases.CASE_A)
    recurrent = ti.Engine.random(cfg, seed=0, dtype="float32", max_tokens=512, max_seqs=2, max_context=128)
    with pytest.raises(ValueError, match="cut back"):
        ti.Draft(recurrent)
