"""Drafts of a few tokens, tested by the model in one step.

A :class:`Draft` is the engine's own model with its matrices in 4 bits, run on the same sequences: a draft's step reads a quarter of the weights. In a
round it continues every sequence by up to ``tokens`` tokens (by no more than its budget leaves), one step each; the sequences are cut back, and the
model runs the drafted tokens through one step of its own, which writes their keys and values over the draft's and gives the logits at every
place. The longest run of drafted tokens that stands is kept, with one token more: at temperature 0 a drafted token stands while it is the model's
own choice, else by the test of ``ops.verify_drafts``, so that every token is distributed as one sampled from the model (not the same token as
without a draft: the uniform numbers are used up in another order). Sequences that cannot be cut back (recurrent states, windows) take no draft.

Over a cache in 8 bits the model is the one that the cache makes of it, and drafts leave a trace there: a page's scale does not shrink while rows are added to it, so the draft's
own rows and those that are cut back may raise it. What of the page's kept rows lies below 2^-6 of the larger scale is then rounded to steps of 2^-9 of it: off by
at most 2^-10 of a scale whose largest value is 224 to 448. Without a draft those rows keep the bits below.
"""
from __future__ import annotations

import copy
from itertools import accumulate
from typing import Callable, Dict, List, Optional, Sequence

import torch

from ..kernels import ops
from ..parts import Linear, Linear4
from ..parts.base import Part, PositionEncoding
from ..sampling import SamplingParams, mix32, sequence_seed
from ..sampling.device import _as_i32

MIXERS, FEED_FORWARDS = ("attention",), ("xielu_mlp", "gelu_mlp", "gated_mlp")


def quantized(model, group: int = 128, zeros: bool = False):
    """A copy of ``model`` that shares everything with it but the matrices of its products, which it has in 4 bits (``parts.Linear4``)."""
    for layer in model.spec.layers:
        if layer.mixer.kind not in MIXERS or (layer.feed_forward is not None and layer.feed_forward.kind not in FEED_FORWARDS):
            raise ValueError(f"a copy in 4 bits is made of layers of {', '.join(MIXERS)} and {', '.join(FEED_FORWARDS)}, not of {layer.mixer.kind} and "
                             f"{layer.feed_forward.kind if layer.feed_forward is not None else 'none'}")
    return with_matrices(model, lambda linear: Linear4(linear, group, zeros))


def with_matrices(model, make: Callable):
    """A copy of ``model`` that shares everything with it but its products, each of which is ``make(product)``."""
    made: Dict[int, object] = {}

    def view(obj):
        if isinstance(obj, (list, tuple)):
            return type(obj)(view(v) for v in obj)
        if isinstance(obj, Linear):
            if id(obj) not in made:
                made[id(obj)] = make(obj)
            return made[id(obj)]
        if isinstance(obj, Part) and not isinstance(obj, PositionEncoding):
            if id(obj) not in made:
                other = made[id(obj)] = copy.copy(obj)
                for name, value in vars(obj).items():
                    setattr(other, name, view(value))
            return made[id(obj)]
        return obj

    other = copy.copy(model)
    other.blocks = []
    for block in model.blocks:
        b = copy.copy(block)
        for name, value in vars(block).items():
            setattr(b, name, view(value))
        other.blocks.append(b)
    other.head = view(model.head)
    return other


class Draft:
    """``tokens``: how many tokens a round drafts at most. ``group``, ``zeros``: see ``parts.Linear4``. ``drafted`` and ``stood`` count the tokens
    that it proposed and those of them that the model kept."""

    def __init__(self, engine, tokens: int = 4, group: int = 128, zeros: bool = False):
        if tokens < 1:
            raise ValueError("a draft has at least one token")
        if any(not g.rolls_back for g in engine.cache.groups) or engine.cache.windowed_groups:
            raise ValueError("a draft needs sequences that can be cut back: no recurrent states and no windows")
        self.engine, self.tokens = engine, int(tokens)
        self.twin = engine.twin(quantized(engine.model, group, zeros))
        self.drafted = self.stood = 0

    def propose(self, slots: Sequence[int], last: Sequence[int], k: int, sampling: SamplingParams, seeds, counters, counts: Optional[Sequence[int]] = None):
        """``k`` tokens for each of ``slots`` (with ``counts`` so many of them for each, at most ``k``), whose last tokens ``last`` the cache does not
        hold yet: (drafts [sequences, k] int32, the probabilities that they were drawn from [sequences, k, vocab], or None for the most likely ones),
        on the device; places beyond a sequence's count hold nothing. The sequences keep their lengths."""
        n, twin = len(slots), self.twin
        lengths = [twin.sequence_length(s) for s in slots]
        steps = torch.zeros(k, n, dtype=torch.int32, device=twin.device)
        q = None if sampling.greedy else torch.empty(k, n, twin.vocab_size, dtype=torch.float32, device=twin.device)
        try:
            rows = []
            for i in range(k):
                before, rows = rows, [r for r in range(n) if counts is None or counts[r] > i]
                ids, at = twin.decode_token_buffer(len(rows)), [slots[r] for r in rows]
                whole = len(rows) == n
                some = None if whole else torch.tensor(rows, dtype=torch.long, device=twin.device)
                if i and rows != before:
                    ids.copy_(steps[i - 1][some])
                logits = twin.decode(at, None if i else [last[r] for r in rows])
                tokens = steps[i] if whole else torch.empty(len(rows), dtype=torch.int32, device=twin.device)
                if sampling.greedy:
                    ops.argmax(logits, tokens, also=ids)
                else:
                    p = q[i] if whole else torch.empty_like(logits)
                    ops.probabilities(p, logits, sampling.temperature, sampling.top_k, sampling.top_p)
                    numbers = (seeds, counters) if whole else (seeds[some], counters[some])
                    ops.sample(logits, tokens, sampling.temperature, sampling.top_k, sampling.top_p, *numbers, also=ids)
                    if not whole:
                        q[i].index_copy_(0, some, p)
                        counters.index_copy_(0, some, numbers[1])
                if not whole:
                    steps[i].index_copy_(0, some, tokens)
        finally:
            for slot, length in zip(slots, lengths):
                twin.truncate(slot, length)
        return steps.t().contiguous(), None if q is None else q.transpose(0, 1)


def _test(engine, logits, drafts, q, sampling: SamplingParams, seeds, counters, counts=None):
    """(how many drafted tokens of each sequence stand, those with the token after them [sequences, k + 1]), on the device. ``counts``: how many
    drafts each sequence has; ``logits`` has k + 1 rows of each all the same."""
    n, k = drafts.shape
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=engine.device)
    accepted = torch.empty(n, dtype=torch.int32, device=engine.device)
    tokens = torch.empty(n, k + 1, dtype=torch.int32, device=engine.device)
    if sampling.greedy:
        chosen = torch.empty(n * (k + 1), dtype=torch.int32, device=engine.device)
        ops.argmax(logits, chosen)
        ops.match_drafts(accepted, tokens, chosen.view(n, k + 1), drafts, counts)
        return accepted, tokens
    p = torch.empty_like(logits)
    ops.probabilities(p, logits, sampling.temperature, sampling.top_k, sampling.top_p)
    u = torch.empty(n, k + 1, dtype=torch.float32, device=engine.device)
    ops.uniforms(u, seeds, counters)
    ops.verify_drafts(accepted, tokens, p.view(n, k + 1, -1), q, drafts, u, counts)
    return accepted, tokens


def decode_batch_drafted(engine, draft: Draft, sampling: SamplingParams, seed: int, live: List[int], slots, logits, results, max_new_tokens: int, stop,
                         on_token: Optional[Callable[[int, int], None]] = None) -> None:
    """As ``generate.decode_batch``, in rounds of a draft and its test: ``live``: the requests in the order of the rows of ``logits`` (those of each one's
    last token so far); ``slots[r]`` is removed, and the sequence freed, when request r ends."""
    from .generate import finished
    device = engine.device
    seeds = _as_i32([sequence_seed(seed, r) for r in live]).to(device)
    draft_seeds = _as_i32([mix32(sequence_seed(seed, r) ^ 0x5BF03635) for r in live]).to(device)       # numbers of its own for the draft
    counters, draft_counters = torch.zeros_like(seeds), torch.zeros_like(seeds)
    first = torch.empty(len(live), dtype=torch.int32, device=device)
    if sampling.greedy:
        ops.argmax(logits, first)
    else:
        ops.sample(logits, first, sampling.temperature, sampling.top_k, sampling.top_p, seeds, counters)
    fresh = [[t] for t in first.tolist()]
    last: Dict[int, int] = {}
    while live:
        rows = []
        for row, r in enumerate(live):
            for token in fresh[row]:
                if token < 0:
                    raise RuntimeError(f"request {r}: the model's probabilities have no weight")
                outcome = finished(token, len(results[r]), max_new_tokens, stop)
                if outcome != "stop":
                    results[r].append(token)
                    if on_token is not None:
                        on_token(r, token)
                if outcome != "go":
                    engine.free_sequence(slots.pop(r))
                    break
            else:
                last[r] = fresh[row][-1]
                rows.append(row)
        if not rows:
            return
        if len(rows) < len(live):
            keep = torch.tensor(rows, dtype=torch.long, device=device)
            seeds, draft_seeds, counters, draft_counters = (t[keep].contiguous() for t in (seeds, draft_seeds, counters, draft_counters))
            live = [live[row] for row in rows]
        at = [slots[r] for r in live]
        lengths = [engine.sequence_length(s) for s in at]
        # A run of c drafts and the token after them ends within a sequence's own budget (and pages, which are set aside for that) and the context.
        counts = [max(0, min(draft.tokens, max_new_tokens - len(results[r]) - 1, engine.max_context - length - 1)) for r, length in zip(live, lengths)]
        k = max(counts)
        tokens = [last[r] for r in live]
        if k < 1:                                            # one token is left to make: a step of its own
            logits = engine.decode(at, tokens)
            first = torch.empty(len(live), dtype=torch.int32, device=device)
            if sampling.greedy:
                ops.argmax(logits, first)
            else:
                ops.sample(logits, first, sampling.temperature, sampling.top_k, sampling.top_p, seeds, counters)
            fresh = [[t] for t in first.tolist()]
            continue
        ragged = min(counts) < k
        drafts, q = draft.propose(at, tokens, k, sampling, draft_seeds, draft_counters, counts if ragged else None)
        runs = [[t] + d[:c] for t, d, c in zip(tokens, drafts.tolist(), counts)]
        logits = engine.step(list(zip(at, runs)), [list(range(c + 1)) for c in counts], few=True)
        if ragged:                                           # k + 1 rows a sequence: its last one again where it has fewer
            ends = list(accumulate(c + 1 for c in counts))
            logits = logits[torch.tensor([end - 1 - max(c - i, 0) for end, c in zip(ends, counts) for i in range(k + 1)], dtype=torch.long, device=device)]
        accepted, kept = _test(engine, logits, drafts, q, sampling, seeds, counters, counts if ragged else None)
        accepted, kept = accepted.tolist(), kept.tolist()
        for slot, length, a in zip(at, lengths, accepted):
            engine.truncate(slot, length + 1 + a)
        draft.drafted += sum(counts)
        draft.stood += sum(accepted)
        fresh = [row[:a + 1] for row, a in zip(kept, accepted)]
