"""Models whose matrices or cache are held in 8 bits: a run of the operators together, as generation uses them.

What the 8-bit cache may change is bounded by running the same model in 32 bits on keys and values that have been through the codes: the engine's logits are held to
those of a plain forward pass in 64 bits with the same codes."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu

# Heads of 64 and 128 (the prompts' tensor-core kernel takes them), and sizes that are no multiple of 128.
HEAD64 = {**helpers.TINY_B, "hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 400, "vocab_size": 500}
HEAD128 = {**helpers.TINY_B, "hidden_size": 192, "num_attention_heads": 4, "num_key_value_heads": 4, "head_dim": 128, "intermediate_size": 272, "vocab_size": 333}


@pytest.fixture(scope="module")
def ti():
    import tileinfer_b200
    return tileinfer_b200


def make(ti, raw, seed=1, **kw):
    from tileinfer_b200.config import ApertusConfig
    cfg = ApertusConfig.from_dict(raw)
    return cfg, ti.Engine.random(cfg, seed=seed, dtype="bfloat16", **{**dict(max_tokens=4096, max_seqs=8, max_context=1024), **kw})


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("raw", [helpers.TINY_B, helpers.TINY_C, HEAD64, HEAD128])
def test_logits_with_an_8_bit_cache(ti, raw):
    """Against the same model with a bfloat16 cache: codes are off by at most 2^-4 of a value, 2.6 % of it on average (the mean of a uniform error of half a step
    over a binade); keys and values carry that to a layer's attention output, which is one of two additions to the stream a layer. Errors are independent: the
    logits stay within a tenth."""
    cfg, plain = make(ti, raw)
    _, engine = make(ti, raw, cache="e4m3")
    prompts = helpers.random_prompts(cfg.vocab_size, [1, 5, 64, 65, 200, 500], 3)
    outs = []
    for e in (plain, engine):
        slots = [e.new_sequence() for _ in prompts]
        logits = [e.step(list(zip(slots, prompts)))]
        for i in range(4):
            logits.append(e.step([(s, [(7 * i + 3) % cfg.vocab_size]) for s in slots]).clone())
        logits.append(e.step([(s, [1, 2, 3]) for s in slots], few=True))
        e.check_health()
        outs.append(torch.cat(logits))
    assert far(outs[1], outs[0]) < 0.1
    assert engine.kv_bytes_per_position() < 0.6 * plain.kv_bytes_per_position()


def test_the_cache_holds_what_the_definition_says(ti):
    """After prompts, single tokens and a cut back: every layer's pages are those that the definition makes of the bfloat16 cache's rows in the same steps,
    as far as the layer's inputs agree: the first layer's, which do not depend on any cache."""
    from numbers8 import same, write
    cfg, plain = make(ti, HEAD64, max_seqs=3)
    _, engine = make(ti, HEAD64, max_seqs=3, cache="e4m3")
    steps = [[list(range(1, 71)), [5, 6], list(range(100, 228))], [[9], [8], [7]], [[3, 4, 5], [1], [2, 2]]]
    slots = [(plain.new_sequence(), engine.new_sequence()) for _ in range(3)]
    held = engine.cache.layer(0)
    k_codes, k_scales = held.k.float().cpu().double(), held.extra[0].cpu().double()
    for tokens in steps:
        for which, e in enumerate((plain, engine)):
            e.step([(s[which], t) for s, t in zip(slots, tokens)])
        table = engine.cache.groups[0].device_table.cpu()
        lens = [engine.sequence_length(s[1]) for s in slots]
        rows, cu = [], [0]
        for (a, b), t, length in zip(slots, tokens, lens):
            pages = plain.cache.groups[0].table(a)
            k = plain.cache.layer(0).k[pages].transpose(1, 2).reshape(-1, 2, 64)[length - len(t):length]
            rows.append(k.cpu())
            cu.append(cu[-1] + len(t))
        k_codes, k_scales = write(k_codes, k_scales, torch.cat(rows), table, [s[1] for s in slots], cu, lens)
        got = engine.cache.layer(0)
        for (_, b), length in zip(slots, lens):
            pages = engine.cache.groups[0].table(b)
            want = k_codes[pages].transpose(1, 2).reshape(-1, 2, 64)[:length]
            assert same(got.k.float().cpu()[pages].transpose(1, 2).reshape(-1, 2, 64)[:length], want)
            assert torch.equal(got.extra[0].cpu().double()[pages], k_scales[pages])
        lengths = [n - 1 if i == 1 and n > 1 else n for i, n in enumerate(lens)]                # the second sequence's last token is written over
        for (a, b), n in zip(slots, lengths):
            plain.truncate(a, n)
            engine.truncate(b, n)


@pytest.mark.parametrize("raw", [helpers.TINY_B, HEAD64])
def test_logits_with_8_bit_weights(ti, raw):
    """Both factors of a product are off by 2.6 % of a value on average: 3.7 % of a sum's size a product, four products a layer, two layers and the head, half of
    it through the stream's additions: the logits stay within a fifth of the bfloat16 model's, and are not the same."""
    cfg, plain = make(ti, raw)
    _, engine = make(ti, raw, weights="e4m3")
    prompts = helpers.random_prompts(cfg.vocab_size, [1, 7, 130], 5)
    outs = []
    for e in (plain, engine):
        slots = [e.new_sequence() for _ in prompts]
        logits = [e.step(list(zip(slots, prompts)))] + [e.step([(s, [i + 1]) for s in slots]).clone() for i in range(3)]
        e.check_health()
        outs.append(torch.cat(logits))
    assert 0 < far(outs[1], outs[0]) < 0.2
    assert engine.weight_bytes() < 0.6 * plain.weight_bytes()


@pytest.mark.parametrize("raw", [helpers.TINY_B, HEAD64, HEAD128])
def test_steps_of_any_cut_and_graphs_agree(ti, raw):
    """Generation (captured steps) picks the tokens of the same engine's steps one by one without graphs; freed pages are used again by other sequences."""
    cfg, engine = make(ti, raw, cache="e4m3", weights="e4m3", max_tokens=1024, max_seqs=4)
    _, other = make(ti, raw, cache="e4m3", weights="e4m3", max_tokens=1024, max_seqs=4, graphs=False)
    prompts = helpers.random_prompts(cfg.vocab_size, [3, 65, 128, 30], 9)
    want = ti.generate(other, prompts, max_new_tokens=70, stop_ids=[])
    for _ in range(2):
        assert ti.generate(engine, prompts, max_new_tokens=70, stop_ids=[]) == want
    assert engine.cache.lengths == {} and all(len(o) == 70 for o in want)
    engine.check_health()


def test_a_draft_of_an_engine_with_an_8_bit_cache(ti):
    raw = {**HEAD64, "intermediate_size": 416}               # a draft's groups of 32 divide it
    cfg, engine = make(ti, raw, cache="e4m3")
    prompts = helpers.random_prompts(cfg.vocab_size, [3, 70], 4)
    draft = ti.Draft(engine, tokens=3, group=32)
    out = ti.generate(engine, prompts, max_new_tokens=40, sampling=ti.SamplingParams(temperature=0.8, top_k=20), seed=3, stop_ids=[], draft=draft)
    assert [len(o) for o in out] == [40, 40] and draft.drafted > 0
    _, e8 = make(ti, raw, weights="e4m3")
    with pytest.raises(ValueError, match="8 bits here"):
        ti.Draft(e8, tokens=2, group=32)


def test_loading(ti, tmp_path):
    from tileinfer_b200.config import config_from_dict
    from tileinfer_b200.weights import write_model_folder
    write_model_folder(config_from_dict(HEAD64), 3, str(tmp_path / "m"))
    model = ti.load_model(str(tmp_path / "m"), max_context=256, max_seqs=2, cache="e4m3", weights="e4m3")
    assert len(ti.generate(model, [5, 17, 3], max_new_tokens=9, stop_ids=[])) == 9
    with pytest.raises(ValueError, match="bfloat16"):
        ti.load_model(str(tmp_path / "m"), dtype="float32", cache="e4m3")


def test_matrices_go_as_their_codes_are_made(ti):
    """Making an engine with 8-bit matrices takes little more memory than the matrices it begins with, and holds half of them."""
    raw = {**helpers.TINY_B, "hidden_size": 1024, "num_attention_heads": 16, "num_key_value_heads": 4, "head_dim": 64, "intermediate_size": 4096, "vocab_size": 512,
           "num_hidden_layers": 8}
    _, plain = make(ti, raw)
    whole = plain.model.weight_bytes()
    del plain
    torch.cuda.empty_cache()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    _, eng = make(ti, raw, weights="e4m3")
    assert eng.model.weight_bytes() < 0.52 * whole
    assert torch.cuda.max_memory_allocated() - base < 1.3 * whole
