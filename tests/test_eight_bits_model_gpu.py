"""Whole models over the 8-bit cache, against a plain pass that reads the engine's own codes, and against what the plain pass would have written.

A step's logits depend on the tokens before it through their keys and values alone. So the last token's pass is repeated plainly, with the codes and scales that stand
in the engine's pages as every layer's keys and values: what is left between the two are roundings of activations to bfloat16. The token's own key and
value are compared with the plain ones: codes are off by 2.6 % of a value in the mean square (half a step over a binade), the activations that they are made
from by another 1 to 2 %."""
import dataclasses
import math
import os

import pytest
import torch

import helpers
import plain_apertus as plain
from test_window_gpu import windowed_architecture

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HEAD128 = {**helpers.TINY_B, "hidden_size": 192, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 128, "intermediate_size": 272, "vocab_size": 333}
MODELS = {"B": helpers.TINY_B, "C": helpers.TINY_C, "D": {**helpers.TINY_D, "num_hidden_layers": 3}, "128": HEAD128}


@pytest.fixture(scope="module")
def ti():
    import tileinfer_b200
    return tileinfer_b200


def make(ti, tmp_path, raw, windows=(), seed=3, **kw):
    """(the plain implementation's view of a model, an engine on it)."""
    from tileinfer_b200.config import ApertusConfig
    from tileinfer_b200.weights import write_model_folder
    raw = {**raw, "max_position_embeddings": 2048}
    config = windowed_architecture().from_dict({**raw, "layer_windows": list(windows)}) if windows else ApertusConfig.from_dict(raw)
    folder = write_model_folder(config, seed, os.path.join(str(tmp_path), "m"))
    pc, w = plain.load_folder(folder)
    return pc, w, ti.Engine.load(folder, dtype="bfloat16", **{**dict(max_context=1024, max_seqs=4, max_tokens=4096, max_step_tokens=128), **kw})


def cached(engine, layer, slot, length):
    """Keys and values [length, heads, dim] as they stand in the pages (zeros where a window's pages were given back)."""
    view = engine.cache.layer(layer)
    table = engine.cache.groups[view.group_index].table(slot)
    out = []
    for pool, scales in zip((view.k, view.v), view.extra):
        heads, _, dim = pool.shape[1:]
        rows = torch.zeros(len(table) * 64, heads, dim)
        for i, page in enumerate(table):
            if page is not None:
                rows[64 * i:64 * (i + 1)] = (pool[page].float() * scales[page][:, None, None]).transpose(0, 1).cpu()
        out.append(rows[:length])
    return out


def last_token(pc, w, token, at, engine, slot, windows=()):
    """Logits of one token at position ``at`` whose layers' keys and values are the engine's, and the layers' own new keys and values."""
    w = {k: (plain.rnd(v, BF16) if v.dim() >= 1 and v.numel() > 1 else v) for k, v in w.items()}
    x, made = plain.embed(w["model.embed_tokens.weight"][:pc.vocab], [token]), []
    for l in range(pc.layers):
        p = f"model.layers.{l}."
        h = plain.rmsnorm(x, w[p + "attention_layernorm.weight"], pc.eps, BF16)
        q, k, v = (plain.linear(h, w[p + f"self_attn.{n}_proj.weight"], BF16).view(1, -1, pc.head_dim) for n in "qkv")
        if pc.qk_norm:
            q, k = (plain.rmsnorm(t, plain.rnd(w[p + f"self_attn.{n}_norm.weight"], BF16), pc.eps, BF16) for t, n in ((q, "q"), (k, "k")))
        cos, sin = plain.rope_tables(pc, torch.tensor([at]), BF16)
        q, k = plain.rope(q, cos, sin, BF16), plain.rope(k, cos, sin, BF16)
        made.append((k[0], v[0]))
        keys, values = cached(engine, l, slot, at + 1)
        o = plain.attention(q, keys, values, 1.0 / math.sqrt(pc.head_dim), BF16, start=at, window=windows[l] if windows else 0)
        x = plain.rnd(x + plain.linear(o.reshape(1, -1), w[p + "self_attn.o_proj.weight"], BF16), BF16)
        h = plain.rmsnorm(x, w[p + "feedforward_layernorm.weight"], pc.eps, BF16)
        x = plain.rnd(x + plain.feed_forward(h, w, p, BF16), BF16)
    h = plain.rmsnorm(x, w["model.norm.weight"], pc.eps, BF16)
    head = w["model.embed_tokens.weight"][:pc.vocab] if pc.tied else w["lm_head.weight"]
    return plain.linear(h, head, BF16)[0], made


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("name", MODELS)
@pytest.mark.parametrize("windows", [(), (0, 100, 37)])
@pytest.mark.parametrize("graphs", [True, False])
def test_steps_against_a_plain_pass_over_the_same_codes(ti, tmp_path, name, windows, graphs):
    """Prompts cut into chunks of 128 tokens, single tokens, runs of a few and of many tokens behind earlier ones."""
    raw = MODELS[name]
    windows = windows[:raw["num_hidden_layers"]]
    pc, w, engine = make(ti, tmp_path, raw, windows, cache="e4m3", graphs=graphs)
    assert engine.cache.layer(0).kind == "paged_kv8" and engine.cache.layer(0).k.dtype == torch.float8_e4m3fn
    tokens = helpers.random_prompts(pc.vocab, [300, 1, 130, 64], 5)
    slots = [engine.new_sequence() for _ in tokens]
    run = lambda new, **kw: engine.step(list(zip(slots, new)), **kw).float().cpu()  # noqa: E731

    def check(logits, seqs):
        for row, i in enumerate(seqs):
            want, made = last_token(pc, w, tokens[i][-1], len(tokens[i]) - 1, engine, slots[i], windows)
            off = float((logits[row] - want).abs().max())
            assert off <= helpers.bf16_logit_tolerance(want), (i, len(tokens[i]), off)
            for l, rows in enumerate(made):
                for mine, got in zip(rows, cached(engine, l, slots[i], len(tokens[i]))):
                    assert far(got[-1], mine) < 0.05, (i, l)

    check(run(tokens), range(4))
    g = torch.Generator().manual_seed(1)
    for step, size in enumerate((1, 1, 3, 1, 200, 1)):
        new = [torch.randint(0, pc.vocab, (size,), generator=g).tolist() for _ in tokens]
        tokens = [t + n for t, n in zip(tokens, new)]
        check(run(new, few=size == 3), range(4) if step in (0, 2, 4, 5) else (0,))
    engine.check_health()


def test_greedy_tokens_with_a_draft_are_the_models_own_choices(ti, tmp_path):
    """Each token, drafted or not, has the largest logit that a pass over the same text gives, but for ties within the roundings of two passes: their activations to bfloat16, and codes
    that flip with them."""
    raw = {**MODELS["D"], "hidden_size": 256, "intermediate_size": 416}              # groups of 32 divide them
    pc, _, engine = make(ti, tmp_path, raw, cache="e4m3")
    prompts = helpers.random_prompts(pc.vocab, [3, 70, 130], 4)
    draft = ti.Draft(engine, tokens=3, group=32)
    outs = [ti.generate(engine, prompts, max_new_tokens=60, stop_ids=[], draft=draft), ti.generate(engine, prompts, max_new_tokens=60, stop_ids=[])]
    assert draft.drafted > 0 and [len(o) for o in outs[0]] == [60] * 3
    for out in outs:
        for prompt, made in zip(prompts, out):
            slot = engine.new_sequence()
            logits = engine.step([(slot, prompt + made[:-1])], [list(range(len(prompt) - 1, len(prompt) + len(made) - 1))]).float().cpu()
            engine.free_sequence(slot)
            short = logits.amax(1) - logits[torch.arange(len(made)), made]
            assert float(short.max()) <= 2 * helpers.bf16_logit_tolerance(logits)
    engine.check_health()


def test_rows_that_are_cut_back_leave_their_scale(ti):
    """A page's scale does not shrink while rows are added to it: what was kept has been rounded to the larger one, which moves nothing but what is below 2^-6 of it, by
    at most half a step of 2^-9."""
    from numbers8 import E4M3, F64, nearest
    from tileinfer_b200.kernels import ops
    nkv, dim, kept = 2, 64, 20
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(64, 2, nkv, dim, generator=g).bfloat16().cuda()
    table, slots = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    found = []
    for size in (1.0, 2.0 ** 12):                            # a run that is kept at its size, one that was large and is cut back
        pools, scales = [torch.zeros(1, nkv, 64, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in "kv"], [torch.ones(1, nkv, device="cuda") for _ in "kv"]

        def write(first, end, by=1.0):
            cu, lens = torch.tensor([0, end - first], dtype=torch.int32).cuda(), torch.tensor([end], dtype=torch.int32).cuda()
            ops.cache_write8(*pools, *scales, rows[first:end, 0] * by, rows[first:end, 1] * by, table, slots, cu, lens, end - first)

        write(0, kept)
        write(kept, kept + 4, size)
        write(kept, kept + 2)
        found.append([(p[0].float().cpu().double(), s[0].cpu().double()) for p, s in zip(pools, scales)])
    for (codes, scale), (moved, larger) in zip(*found):
        assert bool((larger >= 2 ** 10 * scale).all())
        want = nearest(codes[:, :kept] * (scale / larger)[:, None, None])
        assert torch.equal(moved[:, :kept], want)
        value, after = codes[:, :kept] * scale[:, None, None], moved[:, :kept] * larger[:, None, None]
        assert bool(((value == after) | (value.abs() < 2.0 ** -6 * larger[:, None, None])).all())
        assert bool(((value - after).abs() <= 2.0 ** -10 * larger[:, None, None]).all()) and bool((value != after).any())
        assert value.dtype is F64
