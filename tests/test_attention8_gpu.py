"""Attention over pages of 8 bits, against the definition in 64 bits.

Bound of an output o = sum p v: P is rounded to 16 bits (2^-11 of sum p |v| where a run is short, bfloat16's 2^-8 where it is long), o once more
(2^-8 |o|); a score's 32-bit sum over D products is off by at most D 2^-23 scale sum |q k|, which p takes twice (itself and its denominator), with a few
2^-23 more for the exponentials and the scales."""
import pytest
import torch

from numbers8 import E4M3, F64, PAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def make(runs, nq, nkv, dim, seed=0, spoil=True, any_scale=False):
    """runs: (new tokens, length) per sequence. ``spoil``: what no token may see (beyond a sequence's end, unused pages) has the code of NaN."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-length // PAGE) for _, length in runs]
    total, slots = sum(pages) + 3, len(runs) + 2
    order = torch.randperm(total, generator=g)
    table = torch.full((slots, max(pages + [1]) + 1), total - 1, dtype=torch.int32)
    seq_slots = torch.randperm(slots, generator=g)[:len(runs)].to(torch.int32)
    k, v = ((torch.randn(total, nkv, PAGE, dim, generator=g) * 64).clamp(-448, 448).to(E4M3) for _ in range(2))
    scales = [torch.exp2(torch.randint(-8, -4, (total, nkv), generator=g).float()) * ((0.5 + torch.rand(total, nkv, generator=g)) if any_scale else 1.0) for _ in range(2)]
    at, used = 0, torch.zeros(total, PAGE, dtype=torch.bool)
    for slot, n, (_, length) in zip(seq_slots.tolist(), pages, runs):
        table[slot, :n] = order[at:at + n]
        for j in range(n):
            used[order[at + j], :min(PAGE, length - PAGE * j)] = True
        at += n
    if spoil:
        gone = ~used[:, None, :, None].expand_as(k)
        k.view(torch.uint8)[gone], v.view(torch.uint8)[gone] = 0x7F, 0xFF
    cu = torch.tensor([0] + [t for t, _ in runs]).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g).bfloat16()
    return dict(q=q, k=k, v=v, ks=scales[0], vs=scales[1], table=table, seq_slots=seq_slots, cu=cu, lens=torch.tensor([length for _, length in runs], dtype=torch.int32))


def reference(c, scale, window, p_bits):
    """(result, bound), on the device in 64 bits."""
    q, nkv = c["q"].cuda().to(F64), c["k"].shape[1]
    n, nq, dim = q.shape
    group = nq // nkv
    out, bound = torch.zeros(n, nq, dim, dtype=F64, device="cuda"), torch.zeros(n, nq, dim, dtype=F64, device="cuda")
    for b, length in enumerate(c["lens"].tolist()):
        pages = c["table"][int(c["seq_slots"][b]), :-(-length // PAGE)].long()
        first, new = int(c["cu"][b]), int(c["cu"][b + 1] - c["cu"][b])
        key = torch.arange(length, device="cuda")
        for h in range(nkv if new and length else 0):
            keys, values = ((t[pages, h].float().to(F64) * s[pages, h].to(F64)[:, None, None]).reshape(-1, dim)[:length].cuda() for t, s in ((c["k"], c["ks"]), (c["v"], c["vs"])))
            heads = slice(h * group, (h + 1) * group)
            for a in range(0, new, 128):
                t = torch.arange(a, min(a + 128, new), device="cuda")
                last = (length - new + t)[:, None, None]
                hidden = (key > last) | ((key <= last - window) if window else torch.zeros_like(key, dtype=torch.bool))
                qq = q[first + a:first + a + t.numel(), heads]
                p = torch.softmax((qq @ keys.t() * scale).masked_fill(hidden, -torch.inf), -1)
                size = (qq.abs() @ keys.abs().t()).masked_fill(hidden, 0).amax(-1, keepdim=True) * abs(scale) * dim * 2.0 ** -23
                clean = torch.where(torch.isfinite(values), values, 0.0)
                got, rough = p @ clean, p @ clean.abs()
                out[first + a:first + a + t.numel(), heads] = got
                bound[first + a:first + a + t.numel(), heads] = rough * (2.0 ** -p_bits + 2.5 * size + 2.0 ** -17) + got.abs() * 2.0 ** -8
    return out.view(n, nq * dim).cpu(), bound.view(n, nq * dim).cpu()


def call(ops, c, nq, nkv, dim, max_new, window=0, scale=None, **kw):
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.full((c["q"].shape[0] + 1, nq * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention8(out[:-1], d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], scale or dim ** -0.5, nq, nkv, dim, PAGE, max_new,
                   window=window, **kw)
    assert bool((out[-1] == 7).all())
    return out[:-1].cpu()


def check(ops, runs, nq, nkv, dim, window=0, seed=0, max_len=None, any_scale=False, **kw):
    c = make(runs, nq, nkv, dim, seed, any_scale=any_scale)
    new = max([t for t, _ in runs] + [1])
    got = call(ops, c, nq, nkv, dim, new, window, max_len=max_len, **kw)
    long = bool(ops.lib().ti_attention8_widens(len(runs), new, nq, nkv, dim, max_len or PAGE * c["table"].shape[1]))
    want, bound = reference(c, dim ** -0.5, window, 8 if long else 11)
    assert bool(torch.isfinite(got).all())
    off = (got.to(F64) - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())


HEADS = [(4, 2, 16), (6, 3, 32), (2, 2, 48), (16, 4, 64), (5, 1, 80), (12, 2, 96), (3, 3, 112), (32, 8, 128), (16, 1, 128), (8, 2, 256), (2, 1, 208), (40, 1, 64)]


@pytest.mark.parametrize("nq,nkv,dim", HEADS)
@pytest.mark.parametrize("window", [0, 5, 100])
def test_heads_and_runs(ops, nq, nkv, dim, window):
    check(ops, [(1, 1), (3, 64), (4, 65), (0, 70), (8, 200), (2, 129), (5, 5), (7, 1000)], nq, nkv, dim, window, seed=dim)


@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 128, 129, 640, 4097])
@pytest.mark.parametrize("new", [1, 5, 16])
def test_lengths(ops, length, new):
    check(ops, [(min(new, length), length)], 8, 2, 64, seed=length, any_scale=True)


@pytest.mark.parametrize("new", [1, 4, 9, 17, 40])
@pytest.mark.parametrize("group", [1, 3, 4, 8, 20])
def test_rows_of_every_slab_size(ops, new, group):
    check(ops, [(new, 300), (1, 77), (new, new)], 2 * group, 2, 128, seed=group)


@pytest.mark.parametrize("window", [1, 64, 65, 333])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows(ops, window, dim):
    check(ops, [(6, 1500), (6, 7), (3, 64), (16, 700)], 8, 4, dim, window, seed=window)


@pytest.mark.parametrize("seqs", [300, 513, 1030])
def test_many_sequences_of_unequal_lengths(ops, seqs):
    g = torch.Generator().manual_seed(4)
    runs = []
    for _ in range(seqs):
        length = int(torch.randint(1, 300, (1,), generator=g))
        runs.append((int(torch.randint(0, min(length, 6) + 1, (1,), generator=g)), length))
    check(ops, runs, 4, 2, 32)


@pytest.mark.parametrize("nq,nkv,dim", [(32, 8, 128), (4, 1, 64), (2, 2, 256)])
def test_one_long_sequence(ops, nq, nkv, dim):
    check(ops, [(1, 20011)], nq, nkv, dim, any_scale=True)
    check(ops, [(5, 9000), (1, 3)], nq, nkv, dim)


@pytest.mark.parametrize("nq,nkv,dim", [(32, 8, 128), (16, 4, 64), (6, 3, 32), (4, 2, 96), (2, 1, 256), (8, 8, 128), (64, 2, 128)])
@pytest.mark.parametrize("window", [0, 130])
def test_prompts(ops, nq, nkv, dim, window):
    for runs in ([(500, 500)], [(700, 1000), (33, 40), (0, 90), (1, 300), (128, 128)], [(64, 64), (200, 711)]):
        check(ops, runs, nq, nkv, dim, window, seed=dim, any_scale=False)
        check(ops, runs, nq, nkv, dim, window, seed=dim, max_len=1000)


def test_a_long_prompt_in_two_calls(ops):
    check(ops, [(2048, 4096)], 8, 2, 128)
    check(ops, [(1500, 1500), (3, 4000)], 8, 2, 64)


@pytest.mark.parametrize("spread", [0, 10, 60])
def test_scales_of_very_unequal_blocks(ops, spread):
    """Blocks whose scales differ by many powers of two, in keys (a few pages then take all the weight) and values."""
    c = make([(3, 700), (1, 1300)], 8, 2, 128, seed=3)
    g = torch.Generator().manual_seed(spread)
    c["vs"] = torch.exp2(torch.randint(-spread, spread + 1, c["vs"].shape, generator=g).float())
    if spread == 10:
        c["ks"] = torch.exp2(torch.randint(-14, 0, c["ks"].shape, generator=g).float())
    got = call(ops, c, 8, 2, 128, 3)
    want, bound = reference(c, 128 ** -0.5, 0, 11)
    assert bool(((got.to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e4, 1e30])
def test_queries_of_any_size(ops, size):
    c = make([(3, 200)], 8, 2, 64, seed=7)
    c["q"] = (c["q"].float() * size * torch.exp(2 * torch.randn(c["q"].shape, generator=torch.Generator().manual_seed(1)))).bfloat16()
    got = call(ops, c, 8, 2, 64, 3, scale=0.125 / size)
    want, bound = reference(c, 0.125 / size, 0, 11)
    assert bool(((got.to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("window", [0, 20])
def test_zero_queries_over_zero_pages(ops, new, window):
    """The smallest scale times the smallest factor of a row is no 32-bit number; keys that nobody sees stay out all the same."""
    c = make([(new, 70), (new, 40)], 8, 2, 64, seed=3)
    c["q"].zero_(), c["ks"].fill_(2.0 ** -100)
    got = call(ops, c, 8, 2, 64, new, window)
    want, bound = reference(c, 0.125, window, 11)
    assert bool(((got.to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("runs,widened", [([(200, 300), (300, 1500), (1, 64)], True), ([(1, 300), (2, 1500), (0, 900)], False)])
def test_a_sequence_longer_than_was_said_stays_within_its_own(ops, runs, widened):
    """``max_len`` says 512: what the sequence of 1,500 gets is not defined, the others' results are."""
    new = max(t for t, _ in runs)
    assert bool(ops.lib().ti_attention8_widens(3, new, 16, 2, 64, 512)) == widened
    c = make(runs, 16, 2, 64, seed=5)
    got = call(ops, c, 16, 2, 64, new, max_len=512)
    want, bound = reference(c, 0.125, 0, 8)
    right = ((got.to(F64) - want).abs() <= bound).all(-1)
    first, end = int(c["cu"][1]), int(c["cu"][2])
    assert bool(right[:first].all()) and bool(right[end:].all())


def test_nan_codes_reach_the_rows_that_see_them_alone(ops):
    """A NaN value or key of a new token reaches that token and those after it; one before a window's first key nobody."""
    for dim in (64, 128, 48):
        c = make([(6, 300), (4, 40)], 8, 2, dim, seed=dim)
        clean = call(ops, c, 8, 2, dim, 6)
        page = int(c["table"][c["seq_slots"][0], 297 // PAGE])
        for pool, whole in (("v", False), ("k", True)):
            bad = {**c, pool: c[pool].clone()}
            bad[pool].view(torch.uint8)[page, 1, 297 % PAGE, 5] = 0x7F             # position 297: the fourth of tokens 294 to 299
            got, want = call(ops, bad, 8, 2, dim, 6).view(10, 8, dim), clean.view(10, 8, dim)
            assert torch.equal(got[:3], want[:3]) and torch.equal(got[6:], want[6:]) and torch.equal(got[3:6, :4], want[3:6, :4])
            hit = torch.isnan(got[3:6, 4:])
            assert bool(hit.all()) if whole else bool(hit[..., 5].all()) and int(hit.sum()) == 3 * 4
            if not whole:
                keep = [d for d in range(dim) if d != 5]
                assert torch.equal(got[3:6, 4:][..., keep], want[3:6, 4:][..., keep])
    for pool in "kv":
        c = make([(6, 300)], 4, 2, 64, seed=1)
        clean = call(ops, c, 4, 2, 64, 6, window=50)
        page = int(c["table"][c["seq_slots"][0], 3])
        c[pool].view(torch.uint8)[page, :, 244 % PAGE] = 0x7F                     # seen by none: the first token sees 245 to 294
        assert torch.equal(call(ops, c, 4, 2, 64, 6, window=50), clean)
        c[pool].view(torch.uint8)[page, :, 246 % PAGE] = 0x7F                     # seen by the first two
        got = call(ops, c, 4, 2, 64, 6, window=50)
        assert bool(torch.isnan(got[:2]).all()) and torch.equal(got[2:], clean[2:])


def test_nan_and_infinite_queries(ops):
    c = make([(3, 100)], 4, 2, 64, seed=2)
    clean = call(ops, c, 4, 2, 64, 3)
    c["q"][1, 2, 5] = float("nan")
    got, want = call(ops, c, 4, 2, 64, 3).view(3, 4, 64), clean.view(3, 4, 64)
    assert bool(torch.isnan(got[1, 2]).all())
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)


def test_graphs_streams_and_work_spaces(ops):
    """Captured twice with sizes that share their work out differently, replayed in turn on two streams; a caller's work space."""
    cases = [(make([(1, 5000), (2, 70)], 8, 2, 128, seed=1), 2), (make([(300, 300)], 8, 2, 128, seed=2), 300)]
    want = [call(ops, c, 8, 2, 128, t) for c, t in cases]
    for (c, t), w in zip(cases, want):
        seqs, longest = c["lens"].numel(), PAGE * c["table"].shape[1]
        need = ops.attention8_workspace(seqs, t, 8, 2, 128, longest)
        held = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        assert torch.equal(call(ops, c, 8, 2, 128, t, workspace=held), w)
        with pytest.raises(ops.KernelError, match="work space"):
            call(ops, c, 8, 2, 128, t, workspace=held[:need - 1])
    graphs, outs = [], []
    for c, t in cases:
        d = {key: x.cuda() for key, x in c.items()}
        out, graph = torch.zeros(c["q"].shape[0], 8 * 128, dtype=torch.bfloat16, device="cuda"), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attention8(out, d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], 128 ** -0.5, 8, 2, 128, PAGE, t)
        graphs.append((graph, d)); outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out.cpu(), w)


@pytest.mark.parametrize("runs", [[(1, 30000)], [(1, 1000)] * 24, [(5, 3000), (8, 100), (2, 9000)], [(900, 1800)]])
def test_the_same_bits_every_time(ops, runs):
    c = make(runs, 32, 8, 128)
    d = {key: t.cuda() for key, t in c.items()}
    first = None
    for _ in range(40):
        out = torch.full((c["q"].shape[0], 32 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.attention8(out, d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], 128 ** -0.5, 32, 8, 128, PAGE, max(t for t, _ in runs))
        first = out if first is None else first
        assert torch.equal(out, first)
    ops.check_status()


def test_nothing_to_do(ops):
    for runs in ([], [(0, 5), (0, 0)]):
        c = make(runs, 4, 2, 32)
        assert call(ops, c, 4, 2, 32, 1).numel() == 0


def test_refusals(ops):
    c = {key: t.cuda() for key, t in make([(2, 70)], 4, 2, 64).items()}
    out = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    good = dict(out=out, q=c["q"], k_cache=c["k"], v_cache=c["v"], k_scales=c["ks"], v_scales=c["vs"], block_table=c["table"], seq_slots=c["seq_slots"],
                cu_seqlens=c["cu"], kv_lens=c["lens"], scale=0.1, nq=4, nkv=2, head_dim=64, page_size=64, max_new=2)
    ops.attention8(**good)
    for change in (dict(q=c["q"].float()), dict(out=out.float()), dict(k_cache=c["k"].to(torch.bfloat16)), dict(v_cache=c["v"].view(torch.uint8)),
                   dict(k_scales=c["ks"][:-1]), dict(v_scales=c["vs"].bfloat16()), dict(nq=6), dict(nkv=1), dict(head_dim=32), dict(page_size=32), dict(window=-1),
                   dict(block_table=c["table"].long()), dict(cu_seqlens=c["cu"][:1]), dict(kv_lens=c["lens"].cpu()), dict(max_new=-1), dict(scale=0.0), dict(scale=-1.0),
                   dict(max_len=-1), dict(out=out[:1]), dict(q=c["q"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ops.KernelError):
            ops.attention8(**{**good, **change})
    for dim in (24, 272):
        c = {key: t.cuda() for key, t in make([(2, 70)], 1, 1, dim).items()}
        with pytest.raises(ops.KernelError, match="multiple"):
            ops.attention8(torch.zeros(2, dim, dtype=torch.bfloat16, device="cuda"), c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["seq_slots"], c["cu"],
                           c["lens"], 0.1, 1, 1, dim, 64, 2)


@pytest.mark.parametrize("dim", [16, 32, 48, 80, 96, 112, 144, 208, 256])
@pytest.mark.parametrize("window", [0, 300])
def test_prompts_of_every_head_size(ops, dim, window):
    """Sizes whose long runs go through widened pages, and sizes that no prompts' kernel takes."""
    check(ops, [(900, 1000), (0, 70), (300, 300), (1, 64)], 16, 2, dim, window, seed=dim)
    assert bool(ops.lib().ti_attention8_widens(4, 900, 16, 2, dim, 1088)) == (dim <= 128 or dim == 256)
