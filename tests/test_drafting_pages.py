"""A drafted batch stays within the pages that its plan set aside: prompt and budget of every sequence, whatever the others have left.

The cache's books are the real ones, on the CPU; model and draft are stand-ins whose next token is a function of the sequence so far, the draft's
right for some sequences and wrong for others, so that they end at different times."""
from types import SimpleNamespace

import pytest
import torch

from tileinfer_b200.cache import Cache
from tileinfer_b200.engine import drafting
from tileinfer_b200.engine.generate import plan_batches
from tileinfer_b200.parts import CacheRequest
from tileinfer_b200.sampling import SamplingParams

VOCAB, PAGE = 64, 16


def following(history):
    return (sum(history) * 31 + 7 * len(history)) % VOCAB


class Sequences:
    """An engine's side of the loop: steps move the cache's books and give one-hot logits. ``wrong(slot)``: whose tokens it gets wrong."""

    def __init__(self, cache, history, max_context, wrong=lambda slot: False):
        self.cache, self.history, self.max_context, self.wrong = cache, history, max_context, wrong
        self.vocab_size, self.device, self.ids = VOCAB, "cpu", {}

    def sequence_length(self, slot):
        return self.cache.length(slot)

    def truncate(self, slot, length):
        self.cache.truncate(slot, length)
        del self.history[slot][length:]

    def free_sequence(self, slot):
        self.cache.free_slot(slot)

    def step(self, entries, want=None, few=False):
        self.cache.reserve([(s, len(t)) for s, t in entries])
        rows = []
        for i, (slot, tokens) in enumerate(entries):
            assert self.cache.length(slot) + len(tokens) <= self.max_context
            at = [following(self.history[slot] + tokens[:j + 1]) for j in range(len(tokens))]
            rows += [at[j] for j in (want[i] if want is not None else [len(tokens) - 1])]
            self.history[slot] += tokens
            self.cache.advance(slot, len(tokens))
        return torch.nn.functional.one_hot(torch.tensor(rows), VOCAB).float()

    def decode_token_buffer(self, n):
        return self.ids.setdefault(n, torch.zeros(n, dtype=torch.int32))

    def decode(self, slots, tokens=None):
        tokens = self.decode_token_buffer(len(slots)).tolist() if tokens is None else tokens
        logits = self.step([(s, [t]) for s, t in zip(slots, tokens)])
        return torch.stack([row.roll(1) if self.wrong(s) else row for s, row in zip(slots, logits)])


def argmax(logits, out, also=None):
    out.copy_(logits.argmax(1))
    if also is not None:
        also.copy_(out)


def match_drafts(accepted, tokens, chosen, drafts, counts=None):
    for b, row in enumerate(drafts.tolist()):
        count = len(row) if counts is None else int(counts[b])
        a = next((i for i in range(count) if row[i] != int(chosen[b, i])), count)
        accepted[b] = a
        tokens[b] = torch.where(torch.arange(len(row) + 1) <= a, chosen[b], -1)


def drafted(prompts, budget, tokens, wrong, max_tokens, max_context, monkeypatch):
    monkeypatch.setattr(drafting, "ops", SimpleNamespace(argmax=argmax, match_drafts=match_drafts))
    cache = Cache([CacheRequest("paged_kv", kv_heads=1, head_dim=16)], torch.float32, "cpu", max_tokens=max_tokens, max_seqs=len(prompts), page_size=PAGE,
                  max_seq_len=max_context)
    plan = plan_batches([len(p) for p in prompts], budget, len(prompts), max_tokens, PAGE, max_context)
    assert plan.batches == [list(range(len(prompts)))]                   # the plan takes them all at once
    history = {}
    engine = Sequences(cache, history, max_context)
    draft = drafting.Draft.__new__(drafting.Draft)
    draft.engine, draft.tokens, draft.drafted, draft.stood = engine, tokens, 0, 0
    draft.twin = Sequences(cache, history, max_context, wrong)
    slots = {}
    for r in range(len(prompts)):
        slots[r] = cache.alloc_slot()
        history[slots[r]] = []
    results = [[] for _ in prompts]
    logits = engine.step([(slots[r], list(p)) for r, p in enumerate(prompts)])
    drafting.decode_batch_drafted(engine, draft, SamplingParams(), 0, list(range(len(prompts))), slots, logits, results, budget, set())
    assert cache.lengths == {} and cache.free_pages() == cache.num_pages
    return results, draft


def plain(prompt, budget):
    history = list(prompt)
    for _ in range(budget):
        history.append(following(history))
    return history[len(prompt):]


@pytest.mark.parametrize("lengths,budget", [((24, 24), 8), ((40, 8, 23), 8), ((17, 33, 1, 49), 15), ((12, 28), 20), ((31, 31, 31), 1)])
@pytest.mark.parametrize("tokens", [1, 4, 7])
@pytest.mark.parametrize("wrong", [lambda s: s > 0, lambda s: s == 0, lambda s: True, lambda s: False])
def test_unequal_progress_on_a_full_pool(lengths, budget, tokens, wrong, monkeypatch):
    prompts = [[(3 * i + 5 * r) % VOCAB for i in range(n)] for r, n in enumerate(lengths)]
    pool = sum(-(-(n + budget) // PAGE) * PAGE for n in lengths)
    results, draft = drafted(prompts, budget, tokens, wrong, pool, pool, monkeypatch)
    assert results == [plain(p, budget) for p in prompts]
    assert 0 <= draft.stood <= draft.drafted


def test_the_longest_context(monkeypatch):
    """A budget that ends at the longest context, beside a short sequence."""
    prompts = [[1] * 40, [2] * 5]
    results, _ = drafted(prompts, 24, 4, lambda s: s == 1, 96, 64, monkeypatch)
    assert results == [plain(p, 24) for p in prompts]
