"""Tables, ranges and lengths that are wrong, or laid out otherwise: nothing outside them is read or written, and the other sequences get what they should."""
import pytest
import torch

from numbers8 import E4M3, F64, PAGE
from test_attention8_gpu import make, reference

pytestmark = pytest.mark.gpu
SHORT = ([(1, 500), (2, 700), (1, 300)], 8, None)
LONG = ([(200, 500), (300, 700), (100, 300)], 16, 704)            # through widened pages, heads of 64 and of 96
KINDS = [(SHORT, 64), (LONG, 64), (LONG, 96)]


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def run(ops, c, nq, dim, new, longest, table=None, rows=None):
    """The first ``rows`` of q and out are given; what lies behind them in the same memory comes back too."""
    d = {key: t.cuda() for key, t in c.items()}
    rows = c["q"].shape[0] if rows is None else rows
    out = torch.full((c["q"].shape[0] + 70, nq * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    widens = ops.lib().ti_attention8_widens(3, new, nq, 2, dim, longest or PAGE * c["table"].shape[1])
    assert bool(widens) == (longest is not None)
    ops.attention8(out[:rows], d["q"][:rows], d["k"], d["v"], d["ks"], d["vs"], d["table"] if table is None else table, d["seq_slots"], d["cu"], d["lens"], dim ** -0.5, nq, 2, dim,
                   PAGE, new, max_len=longest)
    torch.cuda.synchronize()
    ops.check_status()
    return out.cpu()


def good(got, want, bound, cu, b):
    rows = slice(int(cu[b]), int(cu[b + 1]))
    return bool(((got[rows].to(F64) - want[rows]).abs() <= bound[rows]).all())


@pytest.mark.parametrize("kind,dim", KINDS)
@pytest.mark.parametrize("slot", [-1, -1000, "rows", "rows + 1", 10 ** 6, 2 ** 31 - 1, -2 ** 31])
def test_slots_that_do_not_exist(ops, kind, dim, slot):
    """Their pages read as zeros, so their results are zero. The table stands in a larger one whose rows before and behind it name pages of NaN codes."""
    runs, nq, longest = kind
    new = max(t for t, _ in runs)
    c = make(runs, nq, 2, dim, seed=1)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    cu, table = c["cu"].clone(), c["table"]
    wide = torch.full((table.shape[0] + 4, table.shape[1]), int(c["k"].shape[0]) - 1, dtype=torch.int32)
    wide[2:-2] = table
    c["seq_slots"][1] = {"rows": table.shape[0], "rows + 1": table.shape[0] + 1}.get(slot, slot)
    got = run(ops, c, nq, dim, new, longest, wide.cuda()[2:-2])
    assert good(got, want, bound, cu, 0) and good(got, want, bound, cu, 2)
    assert bool((got[int(cu[1]):int(cu[2])] == 0).all()) and bool((got[int(cu[3]):] == 7).all())


@pytest.mark.parametrize("kind,dim", KINDS)
@pytest.mark.parametrize("end", ["n + 5", 10 ** 6, 2 ** 31 - 1, -3, -2 ** 31])
def test_ranges_beyond_the_rows(ops, kind, dim, end):
    """The last sequence's range ends elsewhere: the sequences before it are right, and nothing behind the rows is written."""
    runs, nq, longest = kind
    new = max(t for t, _ in runs)
    c = make(runs, nq, 2, dim, seed=2)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    cu, n = c["cu"].clone(), c["q"].shape[0]
    c["cu"][3] = n + 5 if end == "n + 5" else end
    got = run(ops, c, nq, dim, new, longest)
    assert good(got, want, bound, cu, 0) and good(got, want, bound, cu, 1)
    assert bool((got[n:] == 7).all())


@pytest.mark.parametrize("kind,dim", KINDS)
def test_fewer_rows_than_the_ranges(ops, kind, dim):
    runs, nq, longest = kind
    new = max(t for t, _ in runs)
    c = make(runs, nq, 2, dim, seed=3)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    rows = int(c["cu"][2]) + 1
    if longest is None:
        rows -= 1                                            # the last sequence has one token
    got = run(ops, c, nq, dim, new, longest, rows=rows)
    assert good(got, want, bound, c["cu"], 0) and good(got, want, bound, c["cu"], 1)
    assert bool((got[rows:] == 7).all())


@pytest.mark.parametrize("kind,dim", KINDS)
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 64, 10 ** 9, 10 ** 5, 0, -1, -64, -1000, -2 ** 31])
def test_lengths_that_cannot_be(ops, kind, dim, length):
    """Longer than a row of the table counts as that, less than nothing as nothing: a sequence without keys gets zeros, in long runs anything."""
    runs, nq, longest = kind
    new = max(t for t, _ in runs)
    c = make(runs, nq, 2, dim, seed=4)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    c["lens"][1] = length
    got = run(ops, c, nq, dim, new, longest)
    cu, n = c["cu"], c["q"].shape[0]
    assert good(got, want, bound, cu, 0) and good(got, want, bound, cu, 2) and bool((got[n:] == 7).all())
    if length <= 0 and longest is None:
        assert bool((got[int(cu[1]):int(cu[2])] == 0).all())


@pytest.mark.parametrize("kind,dim", KINDS)
def test_tables_of_any_pitch(ops, kind, dim):
    """A part of a wider table, rows that overlap, one row whose pitch says nothing; what lies beyond a row's columns is not looked at."""
    runs, nq, longest = kind
    new = max(t for t, _ in runs)
    c = make(runs, nq, 2, dim, seed=5)
    want = run(ops, c, nq, dim, new, longest)
    rows, columns = c["table"].shape
    wide = torch.full((rows, columns + 9), int(c["k"].shape[0]) - 1, dtype=torch.int32)
    wide[:, 4:4 + columns] = c["table"]
    assert torch.equal(run(ops, c, nq, dim, new, longest, wide.cuda()[:, 4:4 + columns]), want)
    one = {**c, "seq_slots": torch.zeros_like(c["seq_slots"])}
    row = c["table"][int(c["seq_slots"][1])].contiguous().cuda()
    want = run(ops, one, nq, dim, new, longest, row[None])
    assert torch.equal(run(ops, one, nq, dim, new, longest, row[:, None].t()), want)              # [1, columns] with strides (1, 1)
    three = {**one, "seq_slots": torch.arange(3, dtype=torch.int32)}
    assert torch.equal(run(ops, three, nq, dim, new, longest, row.expand(3, -1)), want)
    if longest is None:                                      # lengths beyond the columns: the row's next ones name other pages
        c = make(runs, nq, 2, dim, seed=5, spoil=False)
        c["lens"][1] = PAGE * columns
        want = run(ops, c, nq, dim, new, longest)
        c["lens"][1] = PAGE * (columns + 3)
        assert bool(torch.isfinite(want).all()) and torch.equal(run(ops, c, nq, dim, new, longest, wide.cuda()[:, 4:4 + columns]), want)


@pytest.mark.parametrize("written", [1, 3, 100])
def test_writing_through_tables_of_any_pitch(ops, written):
    nkv, dim, seqs, columns = 2, 64, 3, 4
    g = torch.Generator().manual_seed(written)
    table = torch.randperm(seqs * columns, generator=g).to(torch.int32).view(seqs, columns)
    k, v = (torch.randn(seqs * written, nkv, dim, generator=g).bfloat16().cuda() for _ in "kv")
    cu, lens = (torch.arange(seqs + 1) * written).to(torch.int32).cuda(), torch.full((seqs,), written + 60, dtype=torch.int32).cuda()

    def run(table, slots, first=0, seqs=seqs):
        pools = [torch.zeros(12, nkv, PAGE, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in "kv"]
        scales = [torch.ones(12, nkv, device="cuda") for _ in "kv"]
        n = seqs * written
        ops.cache_write8(*pools, *scales, k[:n], v[:n], table, slots, cu[:seqs + 1], lens[:seqs], written)
        return torch.cat([t.view(torch.uint8).flatten().float() for t in pools] + [t.flatten() for t in scales])

    slots = torch.arange(seqs, dtype=torch.int32).cuda()
    want = run(table.cuda(), slots)
    wide = torch.full((seqs, columns + 5), 11, dtype=torch.int32)
    wide[:, 2:2 + columns] = table
    assert torch.equal(run(wide.cuda()[:, 2:2 + columns], slots), want)
    row, zero = table[0].contiguous().cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    want = run(row[None], zero, seqs=1)
    assert bool((want != run(row[None], zero - 1, seqs=1)).any())
    assert torch.equal(run(row[:, None].t(), zero, seqs=1), want)
    assert torch.equal(run(row.expand(5, -1), zero + 4, seqs=1), want)
    # Positions beyond a row's columns are not written, whatever lies behind them.
    lens.fill_(PAGE * columns + 30)
    part = wide.cuda()[:, 2:2 + columns]
    dense = table.cuda()
    assert torch.equal(run(part, slots), run(dense, slots))


def test_runs_longer_than_was_said(ops):
    """``max_new`` says one: what a sequence of 60,000 new tokens gets is not defined, and its work is not counted beyond 32 bits; the others' results are right."""
    nkv, dim, columns, many = 64, 16, 10000, 60000
    c = make([(1, 300), (1, 70)], nkv, nkv, dim, seed=6)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    table = torch.full((c["table"].shape[0], columns), -1, dtype=torch.int32)
    table[:, :c["table"].shape[1]] = c["table"]
    slots = torch.tensor([int(c["seq_slots"][0]), int(c["seq_slots"][1]), int(c["seq_slots"][1])], dtype=torch.int32)
    q = torch.cat([c["q"], torch.zeros(many, nkv, dim, dtype=torch.bfloat16)]).cuda()
    cu, lens = torch.tensor([0, 1, 2, 2 + many], dtype=torch.int32), torch.tensor([300, 70, columns * PAGE], dtype=torch.int32)
    out = torch.full((2 + many + 10, nkv * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention8(out[:2 + many], q, *(c[key].cuda() for key in ("k", "v", "ks", "vs")), table.cuda(), slots.cuda(), cu.cuda(), lens.cuda(), dim ** -0.5, nkv, nkv, dim, PAGE, 1)
    torch.cuda.synchronize()
    ops.check_status()
    assert bool(((out[:2].cpu().to(F64) - want).abs() <= bound).all()) and bool((out[-10:] == 7).all())
