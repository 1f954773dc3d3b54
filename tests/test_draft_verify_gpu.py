"""Probabilities by the sampler's rule and the test of drafted tokens, against plain implementations in 64 bits and whole numbers.

Bound of a probability e / sum e, e = exp((l - max) / T): the quotient's rounding is |argument| 2^-23 of e at most (twice: the difference's and its
own), the exponential and the sum add 2^-20; twice over for the denominator."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


# ------------------------------------------------------------------------------ probabilities
def rule(row, temperature, top_k, top_p):
    """One row in 64 bits: (probabilities, bound)."""
    l = [float("-inf") if math.isnan(v) else v for v in row]
    order = sorted(range(len(l)), key=lambda i: (-l[i], i))
    top = l[order[0]]
    if top == float("-inf"):
        return [0.0] * len(l), [0.0] * len(l)
    e = [1.0 if v == top else math.exp((v - top) / temperature) for v in l]
    kept = order[:top_k] if top_k else order
    if top_p < 1.0:
        total, mass, n = sum(e[i] for i in kept), 0.0, 0
        for n, i in enumerate(kept):
            mass += e[i]
            if mass >= top_p * total:
                break
        kept = kept[:n + 1]
    total, p, bound = sum(e[i] for i in kept), [0.0] * len(l), [0.0] * len(l)
    worst = max([abs((l[i] - top) / temperature) * e[i] for i in kept if 0.0 < e[i] < 1.0] + [0.0]) / total
    for i in kept:
        p[i] = e[i] / total
        arg = abs((l[i] - top) / temperature) if 0.0 < e[i] < 1.0 else 0.0
        bound[i] = p[i] * (2 * (arg + worst * len(kept)) * 2.0 ** -23 + 2.0 ** -19) + 1e-37
    return p, bound


def check_probabilities(ops, x, temperature, top_k=0, top_p=1.0, out=None, logits=None):
    logits = x.cuda() if logits is None else logits
    out = torch.full(x.shape, 5.0, device="cuda") if out is None else out
    ops.probabilities(out, logits, temperature, top_k, top_p)
    got = out.cpu().to(F64)
    for r in range(x.shape[0]):
        want, bound = rule(x[r].to(F64).tolist(), temperature, top_k, top_p)
        want, bound = torch.tensor(want, dtype=F64), torch.tensor(bound, dtype=F64)
        assert bool(((got[r] - want).abs() <= bound).all()), (r, float((got[r] - want).abs().max()))


@pytest.mark.parametrize("vocab", [1, 2, 31, 512, 1023, 4100, 16385, 50257])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 1.7])
def test_probabilities_at_a_temperature(ops, vocab, temperature):
    torch.manual_seed(vocab)
    check_probabilities(ops, torch.randn(3, vocab) * 3, temperature)


@pytest.mark.parametrize("vocab", [5, 512, 5001, 20000])
@pytest.mark.parametrize("top_k", [1, 2, 50, 64, 65, 1000, 4999, 30000])
def test_probabilities_of_the_best(ops, vocab, top_k):
    torch.manual_seed(vocab + top_k)
    check_probabilities(ops, torch.randn(2, vocab) * 2, 0.7, top_k)


@pytest.mark.parametrize("rows", [1, 37, 160, 400])
def test_probabilities_of_many_rows(ops, rows):
    torch.manual_seed(rows)
    x = torch.randn(rows, 40003) * 2
    out = torch.empty_like(x, device="cuda")
    for top_k in (0, 20):
        ops.probabilities(out, x.cuda(), 0.9, top_k)
        z = x.to(F64)
        if top_k:
            z = z.masked_fill(z < z.topk(top_k).values[:, -1:], -math.inf)
        want = torch.softmax(z / 0.9, -1)
        assert bool(((out.cpu().to(F64) - want).abs() <= want * 2.0 ** -17).all())          # arguments up to 20: 2 x 2 x 20 x 2^-23 and 2^-19


def test_probabilities_of_a_large_vocabulary(ops):
    torch.manual_seed(3)
    x = torch.randn(3, 300001) * 2
    for top_k in (0, 7, 250000):
        out = torch.empty_like(x, device="cuda")
        ops.probabilities(out, x.cuda(), 1.1, top_k)
        z = x.to(F64)
        if top_k:
            z = z.masked_fill(z < z.topk(top_k).values[:, -1:], -math.inf)
        want = torch.softmax(z / 1.1, -1)
        assert bool(((out.cpu().to(F64) - want).abs() <= want * 2.0 ** -17).all())


@pytest.mark.parametrize("top_k", [0, 40])
@pytest.mark.parametrize("vocab", [9, 512, 6000])
def test_probabilities_of_a_prefix_by_mass(ops, vocab, top_k):
    """top_p in the middle between two prefixes' masses, so that rounding cannot move it across a border."""
    torch.manual_seed(vocab)
    x = torch.randn(1, vocab) * 2.5
    p, _ = rule(x[0].to(F64).tolist(), 0.8, top_k, 1.0)
    best = sorted(p, reverse=True)
    for n in (0, 1, 3):
        low, high = sum(best[:n]), sum(best[:n + 1])
        check_probabilities(ops, x, 0.8, top_k, float(torch.tensor((low + high) / 2, dtype=torch.float32)))


def test_probabilities_with_ties(ops):
    x = torch.zeros(1, 700)
    x[0, ::7] = 1.0                                           # 100 equal best: the first 40 of them are kept
    check_probabilities(ops, x, 1.0, 40)
    check_probabilities(ops, x, 1.0, 150)
    check_probabilities(ops, torch.zeros(2, 9001), 0.5, 5000)


def test_probabilities_of_masked_rows(ops):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(7, 600)
    x[0, 100:] = -inf
    x[1] = -inf                                               # nothing is left: zeros
    x[2, 5], x[2, 77] = nan, nan
    x[3] = nan
    x[4, 9] = inf                                             # the only one that counts
    x[5, 300:] = torch.finfo(torch.float32).min
    x[6, 1:] = -inf
    for top_k in (0, 3, 200):
        check_probabilities(ops, x, 0.9, top_k)


def test_probabilities_strided(ops):
    torch.manual_seed(8)
    x = torch.randn(4, 1001)
    for shift in (0, 1, 4):
        wide, held = torch.zeros(4, 1030, device="cuda"), torch.full((5, 1031), 3.0, device="cuda")
        wide[:, shift:shift + 1001] = x.cuda()
        check_probabilities(ops, x, 0.6, 12, out=held[:4, shift:shift + 1001], logits=wide[:, shift:shift + 1001])
        assert bool((held[:4, :shift] == 3).all()) and bool((held[:, shift + 1001:] == 3).all()) and bool((held[4] == 3).all())


def test_probabilities_are_what_the_sampler_draws_from(ops):
    torch.manual_seed(9)
    x = (torch.randn(1, 50) * 2).cuda()
    p = torch.empty_like(x)
    ops.probabilities(p, x, 0.8, 20, 0.9)
    rows = 20000
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    ops.sample(x.expand(rows, 50).contiguous(), tokens, 0.8, 20, 0.9, torch.arange(rows, dtype=torch.int32, device="cuda"),
               torch.zeros(rows, dtype=torch.int32, device="cuda"))
    seen = torch.bincount(tokens.long(), minlength=50).to(F64) / rows
    p = p[0].to(F64)
    assert not seen[p == 0].any()
    assert bool(((seen - p).abs() <= 5 * (p * (1 - p) / rows).sqrt() + 1e-9).all())          # five standard deviations


# ------------------------------------------------------------------------------ the test of drafts
def fixed(w):
    return np.rint(np.clip(np.nan_to_num(w, nan=0.0), 0.0, 1.0).astype(np.float64) * 2.0 ** 40).astype(np.int64)


def plain_verify(p, q, drafts, u, counts):
    """Sequence by sequence, in Python's whole numbers."""
    accepted, tokens = [], []
    for b in range(len(drafts)):
        c, a = min(max(int(counts[b]), 0), drafts.shape[1]), 0
        while a < c:
            d = int(drafts[b, a])
            ok = 0 <= d < p.shape[2]
            theirs = np.float32(1.0) if q is None or not ok else q[b, a, d]
            if not np.float32(u[b, a]) * theirs < (p[b, a, d] if ok else np.float32(0.0)):
                break
            a += 1
        row = p[b, a]
        rest = row
        if a < c:
            taken = np.zeros_like(row)
            if q is not None:
                taken = q[b, a]
            elif 0 <= drafts[b, a] < len(row):
                taken[drafts[b, a]] = 1.0
            rest = row - taken
        w = fixed(rest)
        if int(w.sum()) == 0:
            w = fixed(row)
        total, r24 = int(w.sum()), min(int(math.floor(float(u[b, -1]) * 2 ** 24)), 2 ** 24 - 1)
        target = max(1, -(-total * r24 >> 24))
        through = np.cumsum(w)
        token = int(np.searchsorted(through, target)) if total else -1
        accepted.append(a)
        tokens.append(list(drafts[b, :a]) + [token] + [-1] * (drafts.shape[1] - a))
    return np.array(accepted), np.array(tokens)


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def draft_case(seqs, k, vocab, seed, near=0.7):
    rng = np.random.default_rng(seed)
    base = rng.normal(size=(seqs, k + 1, vocab)).astype(np.float32) * 2
    p, q = softmax(base), softmax(base[:, :k] + near * rng.normal(size=(seqs, k, vocab)).astype(np.float32))
    drafts = np.zeros((seqs, k), dtype=np.int32)
    for b in range(seqs):
        for i in range(k):
            drafts[b, i] = min(int(np.searchsorted(np.cumsum(q[b, i].astype(np.float64)), rng.random())), vocab - 1)
    return p, q, drafts, (rng.integers(0, 1 << 24, size=(seqs, k + 1)) / 2.0 ** 24).astype(np.float32), rng.integers(0, k + 1, size=seqs).astype(np.int32)


def run_verify(ops, p, q, drafts, u, counts=None):
    seqs, k = drafts.shape
    accepted = torch.full((seqs,), -7, dtype=torch.int32, device="cuda")
    tokens = torch.full((seqs, k + 1), -7, dtype=torch.int32, device="cuda")
    dev = lambda t: None if t is None else torch.as_tensor(t).cuda()  # noqa: E731
    ops.verify_drafts(accepted, tokens, dev(p), dev(q), dev(drafts), dev(u), dev(counts))
    return accepted.cpu().numpy(), tokens.cpu().numpy()


def check_verify(ops, p, q, drafts, u, counts=None):
    got = run_verify(ops, p, q, drafts, u, counts)
    want = plain_verify(p, q, drafts, u, np.full(len(drafts), drafts.shape[1]) if counts is None else counts)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    return want


@pytest.mark.parametrize("vocab", [1, 2, 33, 512, 1024, 5003, 131072])
@pytest.mark.parametrize("seqs,k", [(1, 0), (1, 4), (5, 1), (9, 7)])
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_verify(ops, vocab, seqs, k, with_q, ragged):
    p, q, drafts, u, counts = draft_case(seqs, k, vocab, vocab + seqs)
    check_verify(ops, p, q if with_q else None, drafts, u, counts if ragged else None)


def test_verify_many_sequences_and_long_runs(ops):
    p, q, drafts, u, counts = draft_case(200, 3, 700, 1)
    accepted, _ = check_verify(ops, p, q, drafts, u, counts)
    assert len(set(accepted.tolist())) == 4                   # every outcome occurs
    p, q, drafts, u, counts = draft_case(3, 70, 64, 2, near=0.05)
    accepted, _ = check_verify(ops, p, q, drafts, u * np.float32(0.9))
    assert accepted.max() > 32


def test_verify_again_and_again(ops):
    """The tickets are left as they were found."""
    for seed in range(4):
        p, q, drafts, u, counts = draft_case(6, 4, 3001, 50 + seed)
        check_verify(ops, p, q, drafts, u)


def test_verify_edges(ops):
    p, q, drafts, u, _ = draft_case(8, 2, 300, 4)
    u[0] = 0.0                                                # accepts whatever the model may say; draws the first token with weight
    u[1] = np.float32(1.0 - 2.0 ** -24)                       # draws the last
    q[2] = p[2, :2]                                           # equal: always accepted
    p[3, 0], q[3, 0] = p[3, 0] * 0 + np.float32(1 / 300), q[3, 0] * 0 + np.float32(1 / 300)
    u[3, 0] = np.float32(1.0 - 2.0 ** -24)
    p[4, 0] = 0.0                                             # the model says nothing: refused, no token
    p[5, 0] = np.nan
    drafts[6, 0], drafts[7, 1] = -1, 300                      # ids outside the vocabulary are refused
    p[7, 0], u[7, 0] = 1.0, 0.5
    want = check_verify(ops, p, q, drafts, u)
    assert want[1][4][0] == -1 and want[1][5][0] == -1 and want[0][6] == 0


def test_verify_where_the_draft_is_nowhere_below(ops):
    """q >= p everywhere (not a distribution, but rounding may come near): the token comes from p."""
    p, q, drafts, u, _ = draft_case(3, 1, 100, 5)
    q[:] = np.maximum(q, p[:, :1]) + np.float32(0.01)
    drafts[:] = 99
    u[:, 0] = 0.999
    p[:, 0, 99] = 0.0
    check_verify(ops, p, q, drafts, u)


def test_verify_strided(ops):
    """A draft's steps lie one after the other ([k, seqs, vocab]), rows with a pitch, addresses that take no wide reads."""
    p, q, drafts, u, _ = draft_case(4, 3, 999, 6)
    want = plain_verify(p, q, drafts, u, np.full(4, 3))
    for shift in (0, 1):
        pd, qd = torch.zeros(4, 4, 1010, device="cuda"), torch.zeros(3, 4, 1017, device="cuda")
        pd[:, :, shift:shift + 999] = torch.as_tensor(p).cuda()
        qd[:, :, shift:shift + 999] = torch.as_tensor(q).cuda().transpose(0, 1)
        accepted, tokens = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, 4, dtype=torch.int32, device="cuda")
        ops.verify_drafts(accepted, tokens, pd[:, :, shift:shift + 999], qd[:, :, shift:shift + 999].transpose(0, 1), torch.as_tensor(drafts).cuda(),
                          torch.as_tensor(u).cuda())
        assert np.array_equal(accepted.cpu().numpy(), want[0]) and np.array_equal(tokens.cpu().numpy(), want[1])


def test_verified_tokens_are_distributed_as_the_models(ops):
    """20,000 runs of one draft each: the first token of the outcome follows p whatever q is (five standard deviations)."""
    rng = np.random.default_rng(7)
    p = np.array([0.5, 0.2, 0.15, 0.1, 0.05], dtype=np.float32)
    q = np.array([0.1, 0.3, 0.1, 0.2, 0.3], dtype=np.float32)
    n = 20000
    drafts = rng.choice(5, size=(n, 1), p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int32)
    u = (rng.integers(0, 1 << 24, size=(n, 2)) / 2.0 ** 24).astype(np.float32)
    pt = torch.as_tensor(p).cuda().expand(n, 2, 5)
    accepted, tokens = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    ops.verify_drafts(accepted, tokens, pt, torch.as_tensor(q).cuda().expand(n, 1, 5), torch.as_tensor(drafts).cuda(), torch.as_tensor(u).cuda())
    seen = np.bincount(tokens[:, 0].cpu().numpy(), minlength=5) / n
    assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def test_verify_on_another_stream_and_in_a_graph(ops):
    p, q, drafts, u, _ = draft_case(5, 3, 4000, 8)
    want = plain_verify(p, q, drafts, u, np.full(5, 3))
    dev = [torch.as_tensor(t).cuda() for t in (p, q, drafts, u)]
    accepted, tokens = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, 4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.verify_drafts(accepted, tokens, *dev)
    side.synchronize()
    assert np.array_equal(tokens.cpu().numpy(), want[1])
    tokens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(accepted, tokens, *dev)
    for _ in range(3):
        tokens.zero_()
        graph.replay()
        assert np.array_equal(tokens.cpu().numpy(), want[1]) and np.array_equal(accepted.cpu().numpy(), want[0])


@pytest.mark.parametrize("seqs,k", [(1, 0), (1, 5), (33, 4), (3, 40)])
def test_match(ops, seqs, k):
    g = torch.Generator().manual_seed(seqs + k)
    chosen = torch.randint(0, 3, (seqs, k + 1), generator=g, dtype=torch.int32)
    drafts = torch.where(torch.rand(seqs, k, generator=g) < 0.8, chosen[:, :k], chosen[:, :k] + 1)
    counts = torch.randint(0, k + 1, (seqs,), generator=g, dtype=torch.int32)
    for c in (None, counts):
        accepted, tokens = torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(seqs, k + 1, dtype=torch.int32, device="cuda")
        ops.match_drafts(accepted, tokens, chosen.cuda(), drafts.cuda(), None if c is None else c.cuda())
        for b in range(seqs):
            a, end = 0, k if c is None else int(c[b])
            while a < end and chosen[b, a] == drafts[b, a]:
                a += 1
            assert int(accepted[b]) == a
            assert tokens[b].tolist() == chosen[b, :a + 1].tolist() + [-1] * (k - a)


def test_uniforms(ops):
    from tileinfer_b200.kernels import library
    seeds = torch.tensor([0, 1, -5, 123456789], dtype=torch.int32, device="cuda")
    counters = torch.tensor([0, 7, -1, 99], dtype=torch.int32, device="cuda")
    out = torch.empty(4, 37, device="cuda")
    ops.uniforms(out, seeds, counters)
    for r, (s, c) in enumerate(((0, 0), (1, 7), (-5, -1), (123456789, 99))):
        want = [library.lib().handle.ti_sampling_uniform((s & 0xFFFFFFFF), (c + i) & 0xFFFFFFFF) for i in range(37)]
        assert out[r].tolist() == want
    assert counters.tolist() == [37, 44, 36, 136]


def test_refusals(ops):
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    base = dict(accepted=i(2), tokens=i(2, 4), p=f(2, 4, 9), q=f(2, 3, 9), drafts=i(2, 3), uniforms=f(2, 4))
    ops.verify_drafts(**base)
    for change in (dict(p=f(2, 3, 9)), dict(p=f(2, 4, 9).double()), dict(p=f(2, 4, 9).cpu()), dict(q=f(2, 3, 8)), dict(q=f(2, 4, 9)), dict(uniforms=f(2, 3)),
                   dict(drafts=i(2, 3).long()), dict(drafts=i(6)), dict(tokens=i(2, 3)), dict(accepted=i(3)), dict(counts=i(3)), dict(counts=f(2)),
                   dict(p=f(2, 9, 4).transpose(1, 2))):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**base, **change})
    for change in (dict(chosen=i(2, 3)), dict(drafts=i(2, 2)), dict(tokens=i(1, 4)), dict(chosen=f(2, 4))):
        with pytest.raises(ops.KernelError):
            ops.match_drafts(**{**dict(accepted=i(2), tokens=i(2, 4), chosen=i(2, 4), drafts=i(2, 3)), **change})
    for args in ((f(2, 9), f(2, 8), 1.0), (f(2, 9), f(2, 9), 0.0), (f(2, 9), f(2, 9), 1.0, -1), (f(2, 9), f(2, 9), 1.0, 0, 0.0), (f(2, 9), f(2, 9).double(), 1.0),
                 (f(9, 2).t(), f(2, 9), 1.0), (f(9), f(9), 1.0)):
        with pytest.raises(ops.KernelError):
            ops.probabilities(*args)
    with pytest.raises(ops.KernelError):
        ops.uniforms(f(2, 3), i(1), i(2))
