"""New rows into pages of 8 bits: codes and scales equal to the definition's, everything else untouched."""
import pytest
import torch

from numbers8 import E4M3, F64, PAGE, power, same, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def pool(pages, heads, dim, seed=0):
    """Any finite codes, scales that differ by block."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(pages, heads, PAGE, dim, generator=g) * 100).clamp(-448, 448).to(E4M3)
    return codes, torch.exp2(torch.randint(-12, 3, (pages, heads), generator=g).float())


def make(runs, heads, dim, dtype=torch.bfloat16, seed=0, spread=2.0):
    """runs: (new rows, length) per sequence."""
    g = torch.Generator().manual_seed(100 + seed)
    need = [-(-length // PAGE) for _, length in runs]
    total, slots = sum(need) + 2, len(runs) + 2
    order, table = torch.randperm(total, generator=g), torch.full((slots, max(need + [1]) + 1), -1, dtype=torch.int32)
    seq_slots = torch.randperm(slots, generator=g)[:len(runs)].to(torch.int32)
    at = 0
    for slot, n in zip(seq_slots.tolist(), need):
        table[slot, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + [t for t, _ in runs]).cumsum(0).to(torch.int32)
    n = int(cu[-1])
    k, v = ((torch.randn(n, heads, dim, generator=g) * torch.exp(spread * torch.randn(n, 1, 1, generator=g))).to(dtype) for _ in range(2))
    (kc, ks), (vc, vs) = pool(total, heads, dim, seed), pool(total, heads, dim, seed + 1)
    return dict(k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs, k=k, v=v, block_table=table, seq_slots=seq_slots, cu_seqlens=cu,
                kv_lens=torch.tensor([length for _, length in runs], dtype=torch.int32))


def on_device(c):
    return {name: t.cuda() for name, t in c.items()}


def expected(c):
    args = c["block_table"], c["seq_slots"].tolist(), c["cu_seqlens"].tolist(), c["kv_lens"].tolist()
    return {kv: write(c[kv + "_cache"].to(F64), c[kv + "_scales"].to(F64), c[kv], *args) for kv in "kv"}


def check(ops, c, max_new):
    d = on_device(c)
    ops.cache_write8(**d, max_new=max_new)
    for kv, (codes, scales) in expected(c).items():
        assert torch.equal(d[kv + "_scales"].cpu().to(F64), scales)
        assert same(d[kv + "_cache"].float().cpu(), codes)
    return d


RUNS = [(1, 1), (1, 64), (1, 65), (0, 70), (3, 66), (64, 128), (65, 129), (1, 1000), (100, 130), (7, 7), (0, 0)]


@pytest.mark.parametrize("heads,dim", [(1, 16), (2, 48), (3, 64), (2, 80), (8, 128), (2, 256), (1, 240)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_runs(ops, heads, dim, dtype):
    check(ops, make(RUNS, heads, dim, dtype, seed=dim), 100)


@pytest.mark.parametrize("new", [1, 2, 63, 64, 65, 300])
@pytest.mark.parametrize("before", [0, 1, 31, 63, 64, 100])
def test_places(ops, new, before):
    check(ops, make([(new, before + new), (min(new, 5), before + 5)], 2, 32, seed=new), new)


def test_max_new_may_be_larger_than_any_run(ops):
    check(ops, make(RUNS, 2, 64), 5000)


def test_one_row_after_another(ops):
    """A page filled row by row, with growing and shrinking rows: the codes that a scale's growth moves are those of the definition."""
    c = make([(1, 1)], 2, 64, seed=5)
    page = int(c["block_table"][c["seq_slots"][0], 0])
    d = on_device(c)
    want = {kv: (c[kv + "_cache"].to(F64), c[kv + "_scales"].to(F64)) for kv in "kv"}
    g = torch.Generator().manual_seed(9)
    for length in range(1, PAGE + 1):
        rows = {kv: (torch.randn(1, 2, 64, generator=g) * 4.0 ** float(torch.randn(1, generator=g))).bfloat16() for kv in "kv"}
        lens = torch.tensor([length], dtype=torch.int32)
        ops.cache_write8(**{**d, "k": rows["k"].cuda(), "v": rows["v"].cuda(), "kv_lens": lens.cuda()}, max_new=1)
        for kv in "kv":
            want[kv] = write(*want[kv], rows[kv], c["block_table"], c["seq_slots"].tolist(), [0, 1], [length])
            assert same(d[kv + "_cache"].float().cpu(), want[kv][0]), length
            assert torch.equal(d[kv + "_scales"].cpu().to(F64), want[kv][1])
    assert float(want["k"][1][page, 0]) > 0


def test_a_page_begins_afresh_and_a_cut_back_run_is_written_over(ops):
    c = make([(5, 10)], 1, 32, seed=2)
    c["k_scales"].fill_(2.0 ** 60)                           # what an earlier sequence left behind
    c["v_scales"].fill_(2.0 ** 60)
    c["cu_seqlens"][1], c["kv_lens"][0] = 5, 5
    d = check(ops, c, 5)
    page = int(c["block_table"][c["seq_slots"][0], 0])
    assert float(d["k_scales"][page, 0]) < 2.0 ** 10
    more = {**{name: t.cpu() for name, t in d.items()}, "k": c["k"][:2] * 1000, "v": c["v"][:2] / 1000, "cu_seqlens": torch.tensor([0, 2], dtype=torch.int32),
            "kv_lens": torch.tensor([5], dtype=torch.int32)}                                   # positions 3 and 4 once more
    check(ops, more, 2)


def test_the_same_call_twice_changes_nothing_more(ops):
    c = make(RUNS, 2, 64, seed=4)
    d = on_device(c)
    ops.cache_write8(**d, max_new=100)
    once = {name: d[name].clone() for name in ("k_scales", "v_scales")}
    codes = {name: d[name].view(torch.uint8).clone() for name in ("k_cache", "v_cache")}
    ops.cache_write8(**d, max_new=100)
    assert all(torch.equal(d[name], t) for name, t in once.items()) and all(torch.equal(d[name].view(torch.uint8), t) for name, t in codes.items())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("first", [0, 1, 8])
def test_rows_inside_wider_ones(ops, dtype, first):
    """Keys and values as parts of a projection's rows, wherever they begin."""
    c = make(RUNS, 2, 64, dtype, seed=6)
    n = c["k"].shape[0]
    d = on_device(c)
    wide = torch.full((n, 300), 3.0, dtype=dtype, device="cuda")
    wide[:, first:first + 128], wide[:, first + 136:first + 264] = d["k"].view(n, 128), d["v"].view(n, 128)
    d["k"], d["v"] = wide[:, first:first + 128].view(n, 2, 64), wide[:, first + 136:first + 264].view(n, 2, 64)
    ops.cache_write8(**d, max_new=100)
    for kv, (codes, scales) in expected(c).items():
        assert same(d[kv + "_cache"].float().cpu(), codes) and torch.equal(d[kv + "_scales"].cpu().to(F64), scales)


def test_heads_in_another_order_and_one_row_for_all(ops):
    c = make([(3, 5)], 4, 32, seed=8)
    c["k"], c["v"] = c["k"].transpose(0, 1).contiguous().transpose(0, 1), c["v"][:1].expand(3, 4, 32)
    d = on_device(c)
    d["k"], d["v"] = c["k"].cuda().transpose(0, 1).contiguous().transpose(0, 1), c["v"][:1].cuda().expand(3, 4, 32)
    ops.cache_write8(**d, max_new=3)
    for kv, (codes, scales) in expected(c).items():
        assert same(d[kv + "_cache"].float().cpu(), codes) and torch.equal(d[kv + "_scales"].cpu().to(F64), scales)


def test_values_at_the_borders(ops):
    c = make([(4, 4), (4, 68), (2, 66)], 2, 32, torch.float32, seed=3)
    k = c["k"]
    k[0], k[1, 0] = 0.0, 448.0
    k[2, 1, :3] = torch.tensor([float("inf"), float("nan"), -float("inf")])
    k[4:8] = float("nan")
    k[8:] = 3.4e38
    c["v"][:4], c["v"][8:] = 2.0 ** -140, 0.0
    d = check(ops, c, 4)
    assert bool((d["k_scales"] >= 2.0 ** -100).all())
    assert float(power(2.0 ** -140)) == 2.0 ** -100


def test_pages_slots_and_lengths_that_do_not_exist_are_left_out(ops):
    c = make([(2, 3), (2, 70), (3, 5), (2, 2), (1, 200)], 2, 32, seed=11)
    before = on_device(c)
    want = expected({**c, "cu_seqlens": torch.tensor([0, 2, 2, 2, 2, 2], dtype=torch.int32)})     # the first sequence alone
    slots = c["seq_slots"]
    c["block_table"][slots[1], 1] = c["k_cache"].shape[0]
    c["kv_lens"][2] = 1                                      # shorter than its run
    slots[3] = c["block_table"].shape[0]
    c["kv_lens"][4] = 64 * c["block_table"].shape[1] + 1     # beyond its row of the table
    d = on_device(c)
    ops.cache_write8(**d, max_new=3)
    for kv, (codes, scales) in want.items():
        assert same(d[kv + "_cache"].float().cpu(), codes) and torch.equal(d[kv + "_scales"].cpu().to(F64), scales)
    assert before["k_cache"].shape == d["k_cache"].shape


def test_captured_and_on_another_stream(ops):
    c = make(RUNS, 2, 64, seed=12)
    want = check(ops, c, 100)
    d, graph = on_device(c), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_write8(**d, max_new=100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    for name in ("k_cache", "v_cache"):
        assert torch.equal(d[name].view(torch.uint8), want[name].view(torch.uint8))
    assert torch.equal(d["k_scales"], want["k_scales"])


def test_nothing_to_write(ops):
    for runs in ([], [(0, 5), (0, 0)]):
        c = make(runs, 2, 32)
        check(ops, c, 1)
        check(ops, c, 0)


def test_refusals(ops):
    d = on_device(make([(2, 3)], 2, 32))
    ops.cache_write8(**d, max_new=2)
    for change in (dict(k=d["k"].half()), dict(v=d["v"].float()), dict(k=d["k"][:, :1]), dict(k=d["k"].cpu()), dict(k_cache=d["k_cache"].view(torch.uint8)),
                   dict(k_scales=d["k_scales"][:, :1]), dict(v_scales=d["v_scales"].double()), dict(block_table=d["block_table"].long()),
                   dict(cu_seqlens=d["cu_seqlens"][:1]), dict(seq_slots=d["seq_slots"].repeat(2)), dict(k=d["k"].transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(v_cache=d["v_cache"][:-1]), dict(max_new=-1), dict(k_cache=d["k_cache"][:, :, :32].contiguous(), v_cache=d["v_cache"][:, :, :32].contiguous()),
                   dict(k_scales=d["k_scales"].t().contiguous().t() if d["k_scales"].shape[0] > 1 else d["k_scales"][:0])):
        with pytest.raises(ops.KernelError):
            ops.cache_write8(**{"max_new": 2, **d, **change})
    for dim in (8, 24, 272):
        d = on_device(make([(2, 3)], 1, dim))
        with pytest.raises(ops.KernelError, match="multiple of 16"):
            ops.cache_write8(**d, max_new=2)
