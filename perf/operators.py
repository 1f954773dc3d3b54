"""The operators of drafting and verifying as cases that can be timed and compared.

A sequence is continued by a draft of a few tokens from weights of 4 bits, which the model itself then tests in one step:

* ``linear4``: y = x Wᵀ for W of 4-bit codes with a scale (and a zero) per group of k. A draft's step and its head. A 32-bit word of ``codes``
  [out, in / 8] holds eight consecutive k: the even ones in its low half, the odd ones in its high half, four bits each in ascending order.
  W[o, k] = (code - zero) * scale with ``scales`` [in / group, out] of x's type and ``zeros`` [in / group, out] uint8, or 8 for all.
* ``attention_few``: the drafted run's attention: a few new tokens of every sequence over the pages of its cache, which hold theirs too.
* ``probabilities``: softmax of logits at a temperature, over the ``top_k`` best (ties to the smaller id).
* ``verify_drafts``: which drafted tokens stand, from the model's and the draft's probabilities and given uniform numbers, and the token
  after them: drawn from what the draft lacks at the first refusal, from the model's own probabilities where none is refused. Weights are
  2^-40 fixed point, so the token does not depend on the order of any sum.

Sizes are those of Apertus-8B and 70B layers (hidden 4,096 / 8,192, 32 or 64 query heads on 8 of 128, feed-forward 21,504, vocabulary 131,072),
of the second tiny configuration of the tests, and what lies between.
"""
import math

import torch

own = False
PAGE = 64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A draft of one user's chat: the up projection, the largest product of a layer, for one token.
        {"name": "draft-up-1", "op": "linear4", "n": 1, "out": 21504, "in": 4096, "group": 128, "zeros": False, "dtype": "bfloat16"},
        # The down projection of a few sequences being drafted together, with a zero per group.
        {"name": "draft-down-8", "op": "linear4", "n": 8, "out": 4096, "in": 21504, "group": 64, "zeros": True, "dtype": "bfloat16"},
        # The head of a large batch: the largest product of all.
        {"name": "draft-head-64", "op": "linear4", "n": 64, "out": 131072, "in": 4096, "group": 128, "zeros": False, "dtype": "bfloat16"},
        # The 32-bit path at the second tiny configuration: the smallest call, where latency is all.
        {"name": "draft-tiny-float32", "op": "linear4", "n": 5, "out": 320, "in": 96, "group": 32, "zeros": True, "dtype": "float32"},
        # One user's chat at the longest context: the run reads the whole cache, which has to be shared out over the GPU.
        {"name": "verify-long-1", "op": "attention", "seqs": 1, "new": 5, "context": 65531, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "ragged": False},
        # A batch of documents of very unequal lengths with runs of unequal lengths; 70B's heads.
        {"name": "verify-ragged-8", "op": "attention", "seqs": 8, "new": 8, "context": 32768, "heads": 64, "kv_heads": 8, "dim": 128, "window": 0,
         "ragged": True},
        # A large batch of short sequences.
        {"name": "verify-batch-64", "op": "attention", "seqs": 64, "new": 4, "context": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "ragged": False},
        # The tokens of one drafted run, at a temperature.
        {"name": "probabilities-5", "op": "probabilities", "rows": 5, "vocab": 131072, "temperature": 0.8, "top_k": 0},
        # The tokens of the runs of a large batch, from the best 50.
        {"name": "probabilities-top-320", "op": "probabilities", "rows": 320, "vocab": 131072, "temperature": 0.7, "top_k": 50},
        # The test of one user's run.
        {"name": "verify-drafts-1", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 131072, "with_q": True, "ragged": False},
        # The test of a large batch's runs, of unequal lengths.
        {"name": "verify-drafts-64", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 131072, "with_q": True, "ragged": True},
        # Drafts that come without probabilities (a greedy draft's), at an odd vocabulary.
        {"name": "verify-greedy-8", "op": "verify", "seqs": 8, "drafts": 7, "vocab": 50257, "with_q": False, "ragged": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear4", "linear4", "attention", "attention", "probabilities", "verify"))
    if op == "linear4":
        group = rng.choice((32, 64, 128))
        k = group * (_log(rng, 128, 21504 - group) // group | 1)          # an odd number of groups: shares of k that do not divide evenly
        out = _log(rng, 100, 32768)
        return {"op": op, "n": _log(rng, 1, 64), "out": out, "in": k, "group": group, "zeros": rng.random() < 0.5,
                "dtype": "float32" if rng.random() < 0.25 and out * k < 1 << 26 else "bfloat16"}
    if op == "attention":
        seqs = _log(rng, 1, 64)
        heads, kv_heads, dim = rng.choice(((32, 8, 128), (64, 8, 128), (16, 4, 64), (6, 3, 32), (4, 2, 16), (12, 2, 96)))
        context = max(16, _log(rng, 16, 131072 // seqs))
        return {"op": op, "seqs": seqs, "new": rng.randint(1, 8), "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "window": rng.choice((0, 0, 0, 200, 1024)), "ragged": rng.random() < 0.5}
    if op == "probabilities":
        vocab = _log(rng, 256, 131072)
        return {"op": op, "rows": _log(rng, 1, 256), "vocab": vocab, "temperature": round(rng.uniform(0.3, 1.5), 2),
                "top_k": rng.choice((0, 0, 1, rng.randint(2, 100), rng.randint(1, vocab)))}
    return {"op": op, "seqs": _log(rng, 1, 64), "drafts": rng.randint(1, 8), "vocab": _log(rng, 256, 131072), "with_q": rng.random() < 0.7,
            "ragged": rng.random() < 0.5}


def _runs(case):
    """(new tokens, positions after them) of every sequence of an attention case: a ragged batch has a sequence without new tokens, too."""
    got = []
    for b in range(case["seqs"]):
        new, length = case["new"], case["context"]
        if case["ragged"]:
            new = 0 if b % 5 == 4 else 1 + (7 * b + new - 1) % new
            length = int(length * (1.0 - 0.618034 * b % 1.0))
        got.append((new, max(length, new)))
    return got


# ---------------------------------------------------------------------------------------------------- what a program has in hand
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _prepare_linear4(case, g):
    dtype, n, out, k, groups = TYPES[case["dtype"]], case["n"], case["out"], case["in"], case["in"] // case["group"]
    codes = torch.zeros(out, k // 8, dtype=torch.int32, device="cuda")
    for i in range(8):                                       # normal weights: the largest of a group meets the code's end
        c = (_normal(g, out, k // 8) * 2.6 + 8).round_().clamp_(0, 15).to(torch.int32)
        codes |= c << (4 * (i // 2) + 16 * (i % 2))
    scales = ((0.8 + 0.4 * torch.rand(groups, out, device="cuda", generator=g)) * 0.0077).to(dtype)
    zeros = torch.randint(5, 12, (groups, out), device="cuda", generator=g).to(torch.uint8) if case["zeros"] else None
    return {"x": _normal(g, n, k).to(dtype), "codes": codes, "scales": scales, "zeros": zeros, "y": torch.empty(n, out, dtype=dtype, device="cuda")}


def _prepare_attention(case, g):
    nq, nkv, dim, runs = case["heads"], case["kv_heads"], case["dim"], _runs(case)
    pages = [-(-length // PAGE) for _, length in runs]
    total, widest, slots = sum(pages), max(pages), len(runs) + 1
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(slots, widest, dtype=torch.int32, device="cuda")
    seq_slots = torch.randperm(slots, device="cuda", generator=g)[:len(runs)].to(torch.int32)
    at = 0
    for slot, n in zip(seq_slots.tolist(), pages):           # pages lie anywhere in the pool
        table[slot, :n] = order[at:at + n]
        at += n
    n = sum(new for new, _ in runs)
    cu = [0]
    for new, _ in runs:
        cu.append(cu[-1] + new)
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"q": _normal(g, n, nq, dim).to(torch.bfloat16), "k": _normal(g, total, nkv, PAGE, dim).to(torch.bfloat16),
            "v": _normal(g, total, nkv, PAGE, dim).to(torch.bfloat16), "table": table, "seq_slots": seq_slots, "cu": int32(cu),
            "kv_lens": int32([length for _, length in runs]), "scale": dim ** -0.5, "new": case["new"], "window": case["window"],
            "out": torch.empty(n, nq * dim, dtype=torch.bfloat16, device="cuda")}


def _logits(g, rows, vocab):
    """Logits as a trained model leaves them: a broad bell and a few tokens well above it."""
    x = _normal(g, rows, vocab) * 2.0
    best = torch.randint(0, vocab, (rows, min(8, vocab)), device="cuda", generator=g)
    return x.scatter_add_(1, best, 9.0 + 2.0 * _normal(g, rows, best.shape[1]))


def _prepare_probabilities(case, g):
    x = _logits(g, case["rows"], case["vocab"])
    return {"logits": x, "temperature": case["temperature"], "top_k": case["top_k"], "out": torch.empty_like(x)}


def _prepare_verify(case, g):
    b, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    logits = _logits(g, b * (k + 1), vocab).view(b, k + 1, vocab)
    p = torch.softmax(logits, -1)
    near = torch.softmax(logits[:, :k].transpose(0, 1) + 0.7 * _normal(g, k, b, vocab), -1)          # a draft step at a time: [k, b, vocab]
    if case["with_q"]:
        drafts = torch.multinomial(near.reshape(k * b, vocab), 1, generator=g).view(k, b).t()
    else:
        drafts = near.argmax(-1).t()
    counts = torch.randint(0, k + 1, (b,), device="cuda", generator=g).to(torch.int32) if case["ragged"] else None
    return {"p": p, "q": near.transpose(0, 1) if case["with_q"] else None, "drafts": drafts.to(torch.int32).contiguous(), "counts": counts,
            "uniforms": (torch.randint(0, 1 << 24, (b, k + 1), device="cuda", generator=g).float() * 2.0 ** -24),
            "accepted": torch.empty(b, dtype=torch.int32, device="cuda"), "tokens": torch.empty(b, k + 1, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    make = {"linear4": _prepare_linear4, "attention": _prepare_attention, "probabilities": _prepare_probabilities, "verify": _prepare_verify}
    return {"op": case["op"], **make[case["op"]](case, _generator(seed))}


# ---------------------------------------------------------------------------------------------------- the plain forms
def _plain_linear4(s):
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device="cuda")
    out, k, groups = s["codes"].shape[0], s["codes"].shape[1] * 8, s["scales"].shape[0]
    code = ((s["codes"][:, :, None] >> shifts) & 15).to(torch.uint8).view(out, groups, k // groups)
    zero = 8.0 if s["zeros"] is None else s["zeros"].t()[:, :, None].float()
    w = ((code.float() - zero) * s["scales"].t()[:, :, None].float()).view(out, k)
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _plain_attention(s):
    (n, nq, dim), nkv, b, new = s["q"].shape, s["k"].shape[1], s["kv_lens"].shape[0], s["new"]
    group, length, cu = nq // nkv, s["kv_lens"].long(), s["cu"].long()
    pages = s["table"][s["seq_slots"].long()].long()
    keys = s["k"][pages].permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, dim).float()
    values = s["v"][pages].permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, dim).float()
    count = cu[1:] - cu[:-1]
    step = torch.arange(new, device="cuda")
    real = step[None, :] < count[:, None]
    rows = torch.where(real, cu[:-1, None] + step[None, :], 0)
    q = s["q"][rows].float().view(b, new, nkv, group, dim).permute(0, 2, 1, 3, 4).reshape(b, nkv, new * group, dim)
    scores = (q @ keys.transpose(-1, -2) * s["scale"]).view(b, nkv, new, group, -1)
    at = (length - count)[:, None] + step[None, :]
    key = torch.arange(keys.shape[2], device="cuda")
    seen = real[:, :, None] & (key <= at[:, :, None])
    if s["window"]:
        seen = seen & (key > at[:, :, None] - s["window"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    weight = e / e.sum(-1, keepdim=True).clamp_min(1e-38)
    o = (weight.view(b, nkv, new * group, -1) @ values).view(b, nkv, new, group, dim).permute(0, 2, 1, 3, 4).reshape(b, new, nq * dim)
    return o[real].to(torch.bfloat16)


def _plain_probabilities(s):
    x, k = s["logits"], s["top_k"]
    e = torch.exp((x - x.amax(-1, keepdim=True)) / s["temperature"])
    if 0 < k < x.shape[1]:
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
        e = e * torch.zeros_like(e).scatter_(1, best, 1.0)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    p, q, drafts, u = s["p"], s["q"], s["drafts"].long(), s["uniforms"]
    b, k = drafts.shape
    count = torch.full((b,), k, device="cuda") if s["counts"] is None else s["counts"].long()
    step = torch.arange(k, device="cuda")
    model = p[:, :k].gather(2, drafts[:, :, None])[:, :, 0]
    draft = torch.ones_like(model) if q is None else q.gather(2, drafts[:, :, None])[:, :, 0]
    stands = (u[:, :k] * draft < model) & (step < count[:, None])
    accepted = stands.long().cumprod(1).sum(1)
    row = torch.arange(b, device="cuda")
    p_row, at = p[row, accepted], accepted.clamp_max(k - 1)
    q_row = torch.zeros_like(p_row).scatter_(1, drafts[row, at][:, None], 1.0) if q is None else q[row, at]
    rest = torch.where((accepted < count)[:, None], (p_row - q_row).clamp_min(0.0), p_row)
    whole = torch.round(rest * 2.0 ** 40).long()
    whole = torch.where((whole.sum(1) == 0)[:, None], torch.round(p_row * 2.0 ** 40).long(), whole)
    through = whole.cumsum(1)
    total, part = through[:, -1], (u[:, k] * 2.0 ** 24).long()
    target = (part * (total >> 24) + ((part * (total & 0xFFFFFF) + 0xFFFFFF) >> 24)).clamp_min(1)
    token = (through < target[:, None]).sum(1)
    place = torch.arange(k + 1, device="cuda")
    padded = torch.cat([drafts, drafts[:, :1]], 1)
    tokens = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], token[:, None], -1))
    return {"accepted": accepted.int(), "tokens": tokens.int()}


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from tileinfer_b200.kernels import ops
    if s["op"] == "linear4":
        ops.linear4(s["y"], s["x"], s["codes"], s["scales"], s["zeros"])
        return s["y"]
    if s["op"] == "attention":
        ops.attention_few(s["out"], s["q"], s["k"], s["v"], s["table"], s["seq_slots"], s["cu"], s["kv_lens"], s["scale"], s["q"].shape[1],
                          s["k"].shape[1], s["q"].shape[2], PAGE, s["new"], window=s["window"])
        return s["out"]
    if s["op"] == "probabilities":
        ops.probabilities(s["out"], s["logits"], s["temperature"], s["top_k"])
        return s["out"]
    ops.verify_drafts(s["accepted"], s["tokens"], s["p"], s["q"], s["drafts"], s["uniforms"], s["counts"])
    return {"accepted": s["accepted"], "tokens": s["tokens"]}


def run(state):
    if own:
        return _own(state)
    plain = {"linear4": _plain_linear4, "attention": _plain_attention, "probabilities": _plain_probabilities, "verify": _plain_verify}
    return plain[state["op"]](state)


def work(case):
    if case["op"] == "linear4":
        n, out, k, size = case["n"], case["out"], case["in"], 2 if case["dtype"] == "bfloat16" else 4
        groups = k // case["group"]
        return {"bytes": out * k // 2 + groups * out * (size + int(case["zeros"])) + n * (k + out) * size, "flops": 2 * n * out * k}
    if case["op"] == "attention":
        nq, nkv, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
        cached = pairs = new_tokens = 0
        for new, length in _runs(case):
            new_tokens += new
            seen = [min(length - new + i + 1, window or length) for i in range(new)]
            pairs += sum(seen)
            cached += min(length, seen[-1] + new - 1) if new else 0          # from the first key that the first new token sees
        return {"bytes": cached * nkv * dim * 4 + new_tokens * nq * dim * 4, "flops": 4 * pairs * nq * dim}
    if case["op"] == "probabilities":
        return {"bytes": case["rows"] * case["vocab"] * 8, "flops": 4 * case["rows"] * case["vocab"]}
    # One row of each side's probabilities a sequence; the draft's is not read where no draft is refused.
    rows = case["seqs"] * case["vocab"]
    return {"bytes": rows * (8 if case["with_q"] else 4) + case["seqs"] * case["drafts"] * 16, "flops": 3 * rows}


# ---------------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def _exact_linear4(s):
    n, (out, words), groups = s["x"].shape[0], s["codes"].shape, s["scales"].shape[0]
    x, k = s["x"].double(), 8 * words
    y = torch.empty(n, out, dtype=torch.float64, device="cuda")
    for a in range(0, out, 8192):
        c = s["codes"][a:a + 8192].long()
        w = torch.empty(c.shape[0], k, dtype=torch.float64, device="cuda")
        for i in range(8):
            w[:, i::8] = ((c >> (4 * (i >> 1) + (16 if i & 1 else 0))) & 0xF).double()
        for j in range(groups):
            part = w[:, j * (k // groups):(j + 1) * (k // groups)]
            part -= s["zeros"][j, a:a + 8192].double()[:, None] if s["zeros"] is not None else 8.0
            part *= s["scales"][j, a:a + 8192].double()[:, None]
        y[:, a:a + 8192] = torch.einsum("nk,ok->no", x, w)
    return y


def _exact_attention(s):
    n, nq, dim = s["q"].shape
    nkv, window = s["k"].shape[1], s["window"]
    got = torch.zeros(n, nq, dim, dtype=torch.float64, device="cuda")
    cu, lens, slots = s["cu"].tolist(), s["kv_lens"].tolist(), s["seq_slots"].tolist()
    for b, length in enumerate(lens):
        pages = s["table"][slots[b], :-(-length // PAGE)].long()
        new = cu[b + 1] - cu[b]
        for h in range(nkv if new else 0):
            keys = s["k"][pages, h].reshape(-1, dim)[:length].double()
            values = s["v"][pages, h].reshape(-1, dim)[:length].double()
            heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            for i in range(new):
                last = length - new + i
                first = max(0, last - window + 1) if window else 0
                z = s["q"][cu[b] + i, heads].double() @ keys[first:last + 1].T * s["scale"]
                got[cu[b] + i, heads] = torch.softmax(z, -1) @ values[first:last + 1]
    return got.view(n, nq * dim)


def _exact_probabilities(s):
    z = s["logits"].double()
    rows, vocab = z.shape
    if 0 < s["top_k"] < vocab:
        # Rank by (value, then smaller id): ids beyond the top_k best lose their logit.
        bar = z.topk(s["top_k"], dim=-1).values[:, -1:]
        above, level = z > bar, z == bar
        keep = above | (level & (level.long().cumsum(-1) <= s["top_k"] - above.sum(-1, keepdim=True)))
        z = z.masked_fill(~keep, -math.inf)
    return torch.softmax(z / s["temperature"], -1)


def exact(case, seed):
    if case["op"] == "verify":
        return None                                          # whole numbers: equal or not
    return {"linear4": _exact_linear4, "attention": _exact_attention, "probabilities": _exact_probabilities}[case["op"]](prepare(case, seed))
