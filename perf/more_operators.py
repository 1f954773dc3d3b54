"""The operators of serving in 8-bit floating point as cases that can be timed and compared.

What a decode step reads most are the weights and the cache. Here both are held as e4m3 codes with 32-bit scales. A block's scale is the smallest
power of two s >= 2^-100 with max |x| <= 448 s over its finite values; its codes are x / s rounded to the nearest (ties to even), NaN for what is not finite.

* ``quantize8``: the codes of a matrix, with a scale for every 128 columns of each row (``rows`` 1: a product's inputs) or of 128 rows (its weights).
* ``linear8``: y = x Wᵀ for W [out, in] in blocks of 128 x 128 and x quantised by row in groups of 128, or given so. Scales lie [in / 128, rows].
* ``cache_write8``: the new keys and values of every sequence into its pages of 64 positions; a block is a page of one head. Rows of the page
  that were there keep their values under a larger scale; a page whose first row is new begins with a new scale.
* ``attention8``: causal attention over such pages, from one new token of a sequence to a prompt's chunk.

Sizes are those of Apertus-8B and 70B layers (hidden 4,096 / 8,192, 32 or 64 query heads on 8 of 128, feed-forward 21,504), of the tiny configurations
of the tests, and what lies between.
"""
import math

import torch

own = False
PAGE, BLOCK, MOST = 64, 128, 448.0
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One user's chat: the up projection, the largest product of a layer, for one token.
        {"name": "up-1", "op": "linear", "n": 1, "out": 21504, "in": 4096, "given": False},
        # A small batch: the down projection, whose rows are long.
        {"name": "down-16", "op": "linear", "n": 16, "out": 4096, "in": 21504, "given": False},
        # The second tiny configuration, five tokens: the smallest call, where latency is all; a last group of less than 128.
        {"name": "tiny-5", "op": "linear", "n": 5, "out": 320, "in": 96, "given": False},
        # A prompt through the up projection, its inputs quantised ahead (another product shares them).
        {"name": "prompt-up-2048", "op": "linear", "n": 2048, "out": 21504, "in": 4096, "given": True},
        # One user's chat at the longest context: one token reads the whole cache, which has to be shared out over the GPU.
        {"name": "cached-long-1", "op": "attention", "seqs": 1, "new": 1, "context": 65536, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "ragged": False},
        # A large batch of short sequences, one token each.
        {"name": "cached-batch-64", "op": "attention", "seqs": 64, "new": 1, "context": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "ragged": False},
        # Documents of very unequal lengths with a few new tokens each (a tested draft), some with none; 70B's heads.
        {"name": "cached-ragged-8", "op": "attention", "seqs": 8, "new": 5, "context": 32768, "heads": 64, "kv_heads": 8, "dim": 128, "window": 0, "ragged": True},
        # The second half of a long prompt that is held in chunks.
        {"name": "cached-prompt-2048", "op": "attention", "seqs": 1, "new": 2048, "context": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "ragged": False},
        # A decode step's keys and values of a large batch: one row into the middle of a page each.
        {"name": "append-64", "op": "write", "seqs": 64, "new": 1, "context": 1000, "kv_heads": 8, "dim": 128, "ragged": False},
        # Prompts of unequal lengths, some of them after earlier positions.
        {"name": "fill-ragged-8", "op": "write", "seqs": 8, "new": 1024, "context": 1500, "kv_heads": 8, "dim": 128, "ragged": True},
        # A layer's inputs, a prompt long.
        {"name": "inputs-2048", "op": "quantize", "n": 2048, "in": 4096, "rows": 1},
        # A weight matrix at load.
        {"name": "weights-down", "op": "quantize", "n": 4096, "in": 21504, "rows": 128},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "attention", "attention", "attention", "write", "quantize"))
    if op == "linear":
        n, k = _log(rng, 1, 2048), 16 * _log(rng, 1, 1344)
        return {"op": op, "n": n, "out": min(_log(rng, 16, 32768), 180388626432 // (n * k)), "in": k, "given": rng.random() < 0.4}
    if op == "attention":
        heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 4, 64), (6, 3, 32), (4, 2, 16), (12, 2, 96)))
        if rng.random() < 0.3:                               # prompts
            seqs, new = rng.randint(1, 4), _log(rng, 33, 1024)
            return {"op": op, "seqs": seqs, "new": new, "context": new + rng.choice((0, rng.randint(1, 1000))), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                    "window": rng.choice((0, 0, 300)), "ragged": rng.random() < 0.5}
        seqs = _log(rng, 1, 64)
        return {"op": op, "seqs": seqs, "new": rng.choice((1, 1, rng.randint(2, 32))), "context": max(32, _log(rng, 32, 131072 // seqs)), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "window": rng.choice((0, 0, 0, 200, 1024)), "ragged": rng.random() < 0.5}
    if op == "write":
        seqs, kv_heads, dim = _log(rng, 1, 64), rng.choice((1, 2, 4, 8)), rng.choice((16, 32, 64, 96, 128, 256))
        new = rng.choice((1, _log(rng, 1, 2048 // seqs)))
        return {"op": op, "seqs": seqs, "new": new, "context": new + _log(rng, 1, 1000) - 1, "kv_heads": kv_heads, "dim": dim, "ragged": rng.random() < 0.5}
    rows = rng.choice((1, 128))
    return {"op": op, "n": _log(rng, 1, 4096), "in": 16 * _log(rng, 1, 1344), "rows": rows}


def _runs(case):
    """(new tokens, positions with them) of every sequence: a ragged batch has a sequence without new tokens, too."""
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


def _scale(largest):
    """The smallest power of two s >= 2^-100 with largest <= 448 s."""
    part, power = torch.frexp(largest)                       # 448 = 0.875 * 2^9
    power = torch.where(largest > 0, power - 9 + (part > 0.875).int(), -100).clamp_min(-100)
    return torch.ldexp(torch.ones_like(largest), power)


def _finite(x):
    return torch.where(torch.isfinite(x), x, 0.0)


def _code(x):
    return torch.where(torch.isfinite(x), x, math.nan).to(E4M3)


def _in_blocks(x, rows):
    """(codes, scales [columns / 128, rows / rows]) of a matrix."""
    n, k = x.shape
    full = torch.nn.functional.pad(x.float(), (0, -k % BLOCK, 0, -n % rows)).view(-(-n // rows), rows, -(-k // BLOCK), BLOCK)
    scale = _scale(_finite(full).abs().amax((1, 3)))
    codes = _code(full / scale[:, None, :, None]).view(torch.uint8).reshape(full.shape[0] * rows, -1)[:n, :k].contiguous().view(E4M3)
    return codes, scale.t().contiguous()


def _inputs(g, n, k):
    """A layer's inputs as they come from a norm: most columns near 1, a few far larger."""
    return (_normal(g, n, k) * (1.0 + 20.0 * (torch.rand(k, device="cuda", generator=g) < 0.01))).to(torch.bfloat16)


def _prepare_linear(case, g):
    n, out, k = case["n"], case["out"], case["in"]
    x = _inputs(g, n, k)
    w = _normal(g, out, k).mul_(0.02)
    codes, scales = _in_blocks(w, BLOCK)
    x, x_scales = _in_blocks(x, 1) if case["given"] else (x, None)
    return {"x": x, "x_scales": x_scales, "codes": codes, "scales": scales, "y": torch.empty(n, out, dtype=torch.bfloat16, device="cuda")}


def _prepare_quantize(case, g):
    n, k, rows = case["n"], case["in"], case["rows"]
    x = _inputs(g, n, k) if rows == 1 else (_normal(g, n, k) * 0.02).to(torch.bfloat16)
    return {"x": x, "rows": rows, "codes": torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(E4M3),
            "scales": torch.zeros(-(-k // BLOCK), -(-n // rows), device="cuda")}


def _pool(g, pages, heads, dim):
    """Pages as they stand in a cache: some blocks' values are larger than others'."""
    x = _normal(g, pages, heads, PAGE, dim) * torch.exp(0.5 * _normal(g, pages, heads, 1, 1))
    scale = _scale(x.abs().amax((2, 3)))
    return x.div_(scale[:, :, None, None]).to(E4M3), scale


def _prepare_paged(case, g):
    runs = _runs(case)
    pages = [-(-length // PAGE) for _, length in runs]
    total, widest, slots = sum(pages), max(pages), len(runs) + 1
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(slots, widest, dtype=torch.int32, device="cuda")
    seq_slots = torch.randperm(slots, device="cuda", generator=g)[:len(runs)].to(torch.int32)
    at = 0
    for slot, n in zip(seq_slots.tolist(), pages):           # pages lie anywhere in the pool
        table[slot, :n] = order[at:at + n]
        at += n
    cu = [0]
    for new, _ in runs:
        cu.append(cu[-1] + new)
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k, k_scales = _pool(g, total, case["kv_heads"], case["dim"])
    v, v_scales = _pool(g, total, case["kv_heads"], case["dim"])
    return {"k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales, "table": table, "seq_slots": seq_slots, "cu": int32(cu),
            "kv_lens": int32([length for _, length in runs]), "new": case["new"]}


def _prepare_attention(case, g):
    n = sum(new for new, _ in _runs(case))
    return {**_prepare_paged(case, g), "q": _normal(g, n, case["heads"], case["dim"]).to(torch.bfloat16), "scale": case["dim"] ** -0.5, "window": case["window"],
            "longest": max(length for _, length in _runs(case)), "out": torch.empty(n, case["heads"] * case["dim"], dtype=torch.bfloat16, device="cuda")}


def _prepare_write(case, g):
    n = sum(new for new, _ in _runs(case))
    row = (n, case["kv_heads"], case["dim"])
    return {**_prepare_paged(case, g), "k_new": (_normal(g, *row) * torch.exp(0.5 * _normal(g, n, 1, 1))).to(torch.bfloat16),
            "v_new": (_normal(g, *row) * torch.exp(0.5 * _normal(g, n, 1, 1))).to(torch.bfloat16)}


def prepare(case, seed):
    make = {"linear": _prepare_linear, "attention": _prepare_attention, "write": _prepare_write, "quantize": _prepare_quantize}
    return {"op": case["op"], **make[case["op"]](case, _generator(seed))}


# ---------------------------------------------------------------------------------------------------- the plain forms
def _widen(codes, scales, rows):
    n, k = codes.shape
    return codes.float() * scales.t().repeat_interleave(rows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_linear(s):
    x, x_scales = _in_blocks(s["x"], 1) if s["x_scales"] is None else (s["x"], s["x_scales"])
    return (_widen(x, x_scales, 1) @ _widen(s["codes"], s["scales"], BLOCK).t()).to(torch.bfloat16)


def _plain_quantize(s):
    codes, scales = _in_blocks(s["x"], s["rows"])
    return {"codes": codes, "scales": scales}


def _plain_attention(s):
    (n, nq, dim), nkv, b, new = s["q"].shape, s["k"].shape[1], s["kv_lens"].shape[0], s["new"]
    group, length, cu = nq // nkv, s["kv_lens"].long(), s["cu"].long()
    pages = s["table"][s["seq_slots"].long()].long()
    keys = (s["k"][pages].float() * s["k_scales"][pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, dim)
    values = (s["v"][pages].float() * s["v_scales"][pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, dim)
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


def _plain_append(s, codes, scales, rows):
    """``rows`` [tokens, heads, dim] into their pages."""
    count = (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count)
    at = s["kv_lens"].long()[seq] - s["cu"][1:].long()[seq] + torch.arange(rows.shape[0], device="cuda")
    pages, place = torch.unique(s["table"][s["seq_slots"].long()[seq], at // PAGE].long(), return_inverse=True)
    m, heads, dim = pages.numel(), rows.shape[1], rows.shape[2]
    fresh = torch.zeros(m, PAGE, heads, dim, device="cuda").index_put_((place, at % PAGE), rows.float()).transpose(1, 2)
    new = torch.zeros(m, PAGE, dtype=torch.bool, device="cuda").index_put_((place, at % PAGE), torch.ones_like(at, dtype=torch.bool))
    first = torch.where(new, torch.arange(PAGE, device="cuda"), PAGE).amin(1)
    kept = torch.arange(PAGE, device="cuda") < first[:, None]
    old, before = codes[pages], scales[pages]
    after = torch.maximum(_scale(_finite(fresh).abs().amax((2, 3))), torch.where(first[:, None] > 0, before, 0.0))
    moved = _code(old.float() * (before / after)[..., None, None]).view(torch.uint8)
    made = _code(fresh / after[..., None, None]).view(torch.uint8)
    got = torch.where(new[:, None, :, None], made, torch.where(kept[:, None, :, None], moved, old.view(torch.uint8)))
    codes.view(torch.uint8).index_copy_(0, pages, got)
    scales.index_copy_(0, pages, after)
    return codes, scales


def _plain_write(s):
    k, k_scales = _plain_append(s, s["k"], s["k_scales"], s["k_new"])
    v, v_scales = _plain_append(s, s["v"], s["v_scales"], s["v_new"])
    return {"k": k, "k_scales": k_scales, "v": v, "v_scales": v_scales}


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from tileinfer_b200.kernels import ops
    if s["op"] == "linear":
        ops.linear8(s["y"], s["x"], s["codes"], s["scales"], s["x_scales"])
        return s["y"]
    if s["op"] == "attention":
        (_, nq, dim), nkv = s["q"].shape, s["k"].shape[1]
        ops.attention8(s["out"], s["q"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["table"], s["seq_slots"], s["cu"], s["kv_lens"], s["scale"], nq, nkv,
                       dim, PAGE, s["new"], window=s["window"], max_len=s["longest"])
        return s["out"]
    if s["op"] == "write":
        ops.cache_write8(s["k"], s["v"], s["k_scales"], s["v_scales"], s["k_new"], s["v_new"], s["table"], s["seq_slots"], s["cu"], s["kv_lens"], s["new"])
        return {"k": s["k"], "k_scales": s["k_scales"], "v": s["v"], "v_scales": s["v_scales"]}
    ops.quantize8(s["codes"], s["scales"], s["x"], s["rows"])
    return {"codes": s["codes"], "scales": s["scales"]}


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "attention": _plain_attention, "write": _plain_write, "quantize": _plain_quantize}[state["op"]](state)


def work(case):
    if case["op"] == "linear":
        n, out, k = case["n"], case["out"], case["in"]
        groups = -(-k // BLOCK)
        inputs = n * (k + 4 * groups) if case["given"] else 2 * n * k
        return {"bytes": out * k + 4 * groups * -(-out // BLOCK) + inputs + 2 * n * out, "flops": 2 * n * out * k}
    if case["op"] == "quantize":
        n, k = case["n"], case["in"]
        return {"bytes": 3 * n * k + 4 * -(-k // BLOCK) * -(-n // case["rows"]), "flops": 2 * n * k}
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "write":
        new = sum(new for new, _ in _runs(case))
        blocks = sum(-(-length // PAGE) - (length - new) // PAGE for new, length in _runs(case) if new)
        return {"bytes": new * row * 6 + blocks * case["kv_heads"] * 16, "flops": 4 * new * row}
    nq, dim, window = case["heads"], case["dim"], case["window"]
    cached = pairs = new_tokens = 0
    for new, length in _runs(case):
        new_tokens += new
        seen = [min(length - new + i + 1, window or length) for i in range(new)]
        pairs += sum(seen)
        cached += min(length, seen[-1] + new - 1) if new else 0              # from the first key that the first new token sees
    return {"bytes": cached * row * 2 + -(-cached // PAGE) * case["kv_heads"] * 8 + new_tokens * nq * dim * 4, "flops": 4 * pairs * nq * dim}


# ---------------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def _exact_power(largest):
    """The scale of blocks whose largest finite value is ``largest`` [...], tried from below."""
    power = torch.floor(torch.log2(largest.clamp_min(1e-300))) - 10
    for _ in range(4):
        power = power + (largest > 448.0 * torch.exp2(power))
    return torch.exp2(power.clamp_min(-100.0))


def _exact_round(v):
    """The nearest number of e4m3: steps of 2^-9 up to 2^-6, then an eighth of the power of two below."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.where(torch.isfinite(v), torch.round(v / step) * step, math.nan)


def _exact_blocks(x, rows):
    n, k = x.shape
    values, scales = torch.empty(n, k, dtype=torch.float64, device="cuda"), torch.empty(-(-k // BLOCK), -(-n // rows), dtype=torch.float64, device="cuda")
    for j in range(scales.shape[0]):
        part = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        row_top = torch.where(torch.isfinite(part), part, 0.0).abs().amax(1)
        top = torch.cat([row_top, row_top.new_zeros(-n % rows)]).view(-1, rows).amax(1)
        scales[j] = _exact_power(top)
        values[:, j * BLOCK:(j + 1) * BLOCK] = _exact_round(part / scales[j].repeat_interleave(rows)[:n, None])
    return values, scales


def _exact_linear(s):
    (out, k), (n, _) = s["codes"].shape, s["x"].shape
    x, x_scales = _exact_blocks(s["x"], 1) if s["x_scales"] is None else (s["x"].double(), s["x_scales"].double())
    y = torch.zeros(n, out, dtype=torch.float64, device="cuda")
    column = torch.arange(out, device="cuda") // BLOCK
    for j in range(x_scales.shape[0]):
        group = slice(j * BLOCK, (j + 1) * BLOCK)
        y += torch.einsum("nk,ok->no", x[:, group] * x_scales[j][:, None], s["codes"][:, group].double() * s["scales"][j].double()[column][:, None])
    return y


def _exact_attention(s):
    n, nq, dim = s["q"].shape
    nkv, window = s["k"].shape[1], s["window"]
    got = torch.zeros(n, nq, dim, dtype=torch.float64, device="cuda")
    cu, lens, slots = s["cu"].tolist(), s["kv_lens"].tolist(), s["seq_slots"].tolist()
    for b, length in enumerate(lens):
        pages = s["table"][slots[b], :-(-length // PAGE)].long()
        new = cu[b + 1] - cu[b]
        key = torch.arange(length, device="cuda")
        for h in range(nkv if new else 0):
            keys = (s["k"][pages, h].double() * s["k_scales"][pages, h].double()[:, None, None]).reshape(-1, dim)[:length]
            values = (s["v"][pages, h].double() * s["v_scales"][pages, h].double()[:, None, None]).reshape(-1, dim)[:length]
            heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            for a in range(0, new, 64):
                last = length - new + torch.arange(a, min(new, a + 64), device="cuda")
                z = torch.einsum("thd,kd->thk", s["q"][cu[b] + a:cu[b] + min(new, a + 64), heads].double(), keys) * s["scale"]
                hidden = (key > last[:, None]) | ((key <= last[:, None] - window) if window else False)
                got[cu[b] + a:cu[b] + min(new, a + 64), heads] = torch.softmax(z.masked_fill(hidden[:, None, :], -math.inf), -1) @ values
    return got.view(n, nq * dim)


def _exact_append(s, codes, scales, rows):
    got, power = codes.double(), scales.double()
    cu, lens, slots = s["cu"].tolist(), s["kv_lens"].tolist(), s["seq_slots"].tolist()
    for b, length in enumerate(lens):
        new = cu[b + 1] - cu[b]
        at = length - new
        while at < length:                                   # one page after another
            first, end, page = at % PAGE, min(length - at // PAGE * PAGE, PAGE), int(s["table"][slots[b], at // PAGE])
            token = cu[b] + at - (length - new)
            x = rows[token:token + end - first].double().transpose(0, 1)
            scale = _exact_power(torch.where(torch.isfinite(x), x, 0.0).abs().amax((1, 2)))
            if first:
                scale = torch.maximum(scale, power[page])
                got[page, :, :first] = _exact_round(got[page, :, :first] * (power[page] / scale)[:, None, None])
            got[page, :, first:end] = _exact_round(x / scale[:, None, None])
            power[page] = scale
            at += end - first
    return got, power


def _exact_write(s):
    (k, k_scales), (v, v_scales) = (_exact_append(s, s[c], s[c + "_scales"], s[c + "_new"]) for c in "kv")
    return {"k": k, "k_scales": k_scales, "v": v, "v_scales": v_scales}


def _exact_quantize(s):
    values, scales = _exact_blocks(s["x"], s["rows"])
    return {"codes": values, "scales": scales}


def exact(case, seed):
    return {"linear": _exact_linear, "attention": _exact_attention, "write": _exact_write, "quantize": _exact_quantize}[case["op"]](prepare(case, seed))
