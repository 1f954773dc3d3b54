"""Attention of a few new tokens of every sequence over the paged cache, against the definition in 64 bits.

Bound of an output o = sum p v: P is rounded to bfloat16 (2^-8 of sum p |v|), o once more (2^-8 |o|); a score's 32-bit sum over D products is off by
at most D 2^-23 scale sum |q k|, which p takes twice (itself and its denominator), with a few 2^-23 more for the exponentials."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
PAGE = 64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def make(runs, nq, nkv, dim, seed=0, spoil=False):
    """runs: (new tokens, length) per sequence. ``spoil``: what no token may see (beyond a sequence's end, unused pages) is NaN."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-length // PAGE) for _, length in runs]
    total, slots = sum(pages) + 3, len(runs) + 2
    order = torch.randperm(total, generator=g)
    table = torch.full((slots, max(pages + [1]) + 1), total - 1 if total else 0, dtype=torch.int32)
    seq_slots = torch.randperm(slots, generator=g)[:len(runs)].to(torch.int32)
    k, v = torch.randn(total, nkv, PAGE, dim, generator=g).bfloat16(), torch.randn(total, nkv, PAGE, dim, generator=g).bfloat16()
    at, used = 0, torch.zeros(total, PAGE, dtype=torch.bool)
    for slot, n, (_, length) in zip(seq_slots.tolist(), pages, runs):
        table[slot, :n] = order[at:at + n]
        for j in range(n):
            used[order[at + j], :min(PAGE, length - PAGE * j)] = True
        at += n
    if spoil:
        gone = ~used[:, None, :, None].expand_as(k)
        k[gone], v[gone] = float("nan"), float("inf")
    cu = torch.tensor([0] + [t for t, _ in runs]).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g).bfloat16()
    return dict(q=q, k=k, v=v, table=table, seq_slots=seq_slots, cu=cu, lens=torch.tensor([length for _, length in runs], dtype=torch.int32))


def reference(c, scale, window):
    """(result, bound), token by token."""
    q, nkv = c["q"].to(F64), c["k"].shape[1]
    n, nq, dim = q.shape
    out, bound = torch.zeros(n, nq, dim, dtype=F64), torch.zeros(n, nq, dim, dtype=F64)
    for b, length in enumerate(c["lens"].tolist()):
        pages = c["table"][int(c["seq_slots"][b]), :-(-length // PAGE)].long()
        first, new = int(c["cu"][b]), int(c["cu"][b + 1] - c["cu"][b])
        for h in range(nq):
            keys = c["k"][pages, h // (nq // nkv)].reshape(-1, dim)[:length].to(F64)
            values = c["v"][pages, h // (nq // nkv)].reshape(-1, dim)[:length].to(F64)
            for i in range(new):
                end = length - new + i + 1
                start = max(0, end - window) if window else 0
                if end <= 0:
                    continue
                kk, vv, qq = keys[start:end], values[start:end], q[first + i, h]
                p = torch.softmax(kk @ qq * scale, 0)
                rough = float((kk.abs() @ qq.abs()).max()) * abs(scale) * dim * 2.0 ** -23
                out[first + i, h] = p @ vv
                bound[first + i, h] = (p @ vv.abs()) * (2.0 ** -8 + 2.5 * rough + 2.0 ** -18) + out[first + i, h].abs() * 2.0 ** -8
    return out.view(n, nq * dim), bound.view(n, nq * dim)


def call(ops, c, nq, nkv, dim, max_new, window=0, scale=None, **kw):
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.full((c["q"].shape[0], nq * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention_few(out, d["q"], d["k"], d["v"], d["table"], d["seq_slots"], d["cu"], d["lens"], scale or dim ** -0.5, nq, nkv, dim, PAGE, max_new,
                      window=window, **kw)
    return out.cpu()


def check(ops, runs, nq, nkv, dim, window=0, seed=0, spoil=True):
    c = make(runs, nq, nkv, dim, seed, spoil)
    got = call(ops, c, nq, nkv, dim, max([t for t, _ in runs] + [1]), window)
    want, bound = reference(c, dim ** -0.5, window)
    assert bool(torch.isfinite(got).all())
    off = (got.to(F64) - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())


HEADS = [(4, 2, 16), (6, 3, 32), (2, 2, 48), (16, 4, 64), (5, 1, 80), (12, 2, 96), (3, 3, 112), (32, 8, 128), (16, 1, 128), (8, 2, 256)]


@pytest.mark.parametrize("nq,nkv,dim", HEADS)
@pytest.mark.parametrize("window", [0, 5, 100])
def test_heads_and_runs(ops, nq, nkv, dim, window):
    check(ops, [(1, 1), (3, 64), (4, 65), (0, 70), (8, 200), (2, 129), (5, 5), (7, 1000)], nq, nkv, dim, window, seed=dim)


@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 128, 129, 640, 4097])
@pytest.mark.parametrize("new", [1, 5, 16])
def test_lengths(ops, length, new):
    check(ops, [(min(new, length), length)], 8, 2, 64, seed=length)


@pytest.mark.parametrize("new", [1, 4, 9, 17, 40])
@pytest.mark.parametrize("group", [1, 3, 4, 8, 20])
def test_rows_of_every_slab_size(ops, new, group):
    """Rows (new tokens x heads per KV head) from one to several slabs of 64."""
    check(ops, [(new, 300), (1, 77), (new, new)], 2 * group, 2, 64, seed=group)


@pytest.mark.parametrize("window", [1, 64, 65, 333])
def test_windows(ops, window):
    check(ops, [(6, 1500), (6, 7), (3, 64), (16, 700)], 8, 4, 128, window, seed=window)


@pytest.mark.parametrize("seqs", [300, 513, 1030])
def test_many_sequences_of_unequal_lengths(ops, seqs):
    g = torch.Generator().manual_seed(4)
    runs = []
    for _ in range(seqs):
        length = int(torch.randint(1, 300, (1,), generator=g))
        runs.append((int(torch.randint(0, min(length, 6) + 1, (1,), generator=g)), length))
    check(ops, runs, 4, 2, 32)


def test_one_long_sequence(ops):
    check(ops, [(5, 40000)], 8, 2, 128)


def test_a_sequence_shorter_than_its_run_and_empty_ones(ops):
    """A length that does not reach the run (nothing a step makes): tokens before the start see nothing and get zeros."""
    check(ops, [(4, 2), (3, 0), (2, 10)], 4, 2, 64)
    c = make([(3, 0)], 4, 2, 64)
    assert not call(ops, c, 4, 2, 64, 3).any()
    c = make([(0, 5), (0, 0)], 4, 2, 64)
    call(ops, c, 4, 2, 64, 0)


def test_sharp_scores(ops):
    """Scores of a few hundred: a maximum that moves by tens from tile to tile."""
    c = make([(4, 777)], 4, 1, 64, 6)
    c["q"] = (c["q"].float() * 24).bfloat16()
    got = call(ops, c, 4, 1, 64, 4)
    want, bound = reference(c, 64 ** -0.5, 0)
    assert bool(((got.to(F64) - want).abs() <= bound).all())


def test_one_new_token_equals_decode_attention_within_the_bound(ops):
    check(ops, [(1, 999), (1, 64), (1, 1)], 32, 8, 128)


def test_own_workspace_other_stream_and_graph(ops):
    runs = [(5, 900), (2, 31), (0, 3), (5, 4000)]
    c = make(runs, 16, 4, 128, 3)
    d = {key: t.cuda() for key, t in c.items()}
    args = (d["q"], d["k"], d["v"], d["table"], d["seq_slots"], d["cu"], d["lens"], 128 ** -0.5, 16, 4, 128, PAGE, 5)
    want = torch.empty(12, 16 * 128, dtype=torch.bfloat16, device="cuda")
    ops.attention_few(want, *args)
    ws = torch.empty(ops.attention_few_workspace(4, 5, 16, 4, 128), dtype=torch.uint8, device="cuda")
    got = torch.zeros_like(want)
    ops.attention_few(got, *args, workspace=ws)
    assert torch.equal(got, want)                              # the same bits every time
    side, got = torch.cuda.Stream(), torch.zeros_like(want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_few(got, *args)
    side.synchronize()
    assert torch.equal(got, want)
    graph, got = torch.cuda.CUDAGraph(), torch.zeros_like(want)
    with torch.cuda.graph(graph):
        ops.attention_few(got, *args, workspace=ws)
    d["lens"][3] = 1000                                        # a captured call reads the lengths of its replay
    c["lens"][3] = 1000
    graph.replay()
    ref, bound = reference(c, 128 ** -0.5, 0)
    assert bool(((got.cpu().to(F64) - ref).abs() <= bound).all())


def test_refusals(ops):
    c = make([(2, 70)], 4, 2, 64)
    d = {key: t.cuda() for key, t in c.items()}
    base = dict(out=torch.empty(2, 256, dtype=torch.bfloat16, device="cuda"), q=d["q"], k_cache=d["k"], v_cache=d["v"], block_table=d["table"],
                seq_slots=d["seq_slots"], cu_seqlens=d["cu"], kv_lens=d["lens"], scale=0.1, nq=4, nkv=2, head_dim=64, page_size=64, max_new=2)
    ops.attention_few(**base)
    ws = torch.empty(16, dtype=torch.uint8, device="cuda")
    for change in (dict(q=d["q"].float()), dict(q=d["q"].cpu()), dict(out=base["out"][:1]), dict(nkv=3), dict(nq=6), dict(head_dim=32), dict(page_size=32),
                   dict(kv_lens=d["lens"].long()), dict(cu_seqlens=d["cu"][:1]), dict(seq_slots=d["table"][0]), dict(workspace=ws), dict(window=-1), dict(scale=0.0), dict(scale=-1.0),
                   dict(v_cache=d["v"][:1]), dict(max_new=-1), dict(q=d["q"].transpose(0, 1).contiguous().transpose(0, 1)), dict(block_table=d["table"][0])):
        with pytest.raises(ops.KernelError):
            ops.attention_few(**{**base, **change})
    odd = make([(2, 70)], 4, 2, 24)
    with pytest.raises(ops.KernelError):                       # a head size without an instance
        call(ops, odd, 4, 2, 24, 2)
