"""The 8-bit operators as programs call them: together, from several threads, counted, with tables and lengths that are wrong."""
import threading

import pytest
import torch

from numbers8 import E4M3, F64, PAGE
from test_attention8_gpu import make, reference
from test_drafting_launches_gpu import kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def product(ops, n, out, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    w, x = torch.randn(out, k, generator=g).bfloat16().cuda(), torch.randn(n, k, generator=g).bfloat16().cuda()
    codes, scales = torch.empty(out, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(-(-k // 128), -(-out // 128), device="cuda")
    ops.quantize8(codes, scales, w, 128)
    y = torch.empty(n, out, dtype=torch.bfloat16, device="cuda")
    return lambda: ops.linear8(y, x, codes, scales), y


def attention(ops, runs, nq=8, nkv=2, dim=64, seed=0, **kw):
    c = make(runs, nq, nkv, dim, seed=seed)
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.empty(c["q"].shape[0], nq * dim, dtype=torch.bfloat16, device="cuda")
    new = max(t for t, _ in runs)
    return lambda: ops.attention8(out, d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], dim ** -0.5, nq, nkv, dim, PAGE, new, **kw), out


CASES = {"few": lambda ops, s: product(ops, 3 + s, 640, 512, s), "mid": lambda ops, s: product(ops, 10 + s, 640, 512, s), "many": lambda ops, s: product(ops, 700 + s, 4096, 512, s),
         "short": lambda ops, s: attention(ops, [(1, 900 + s), (2, 5000), (1, 64)], seed=s), "long": lambda ops, s: attention(ops, [(400 + s, 900), (300, 300)], 16, seed=s)}


@pytest.mark.parametrize("kind", CASES)
def test_two_threads_on_one_stream(ops, kind):
    cases = [CASES[kind](ops, seed) for seed in (1, 2, 3)]
    want = []
    for call, out in cases:
        call()
        want.append(out.clone())
    wrong, start = [], threading.Barrier(len(cases))

    def work(i):
        call, out = cases[i]
        start.wait()
        for _ in range(20):
            seen = []
            for _ in range(10):
                call()
                seen.append(out.clone())
            wrong.extend(i for got in seen if not torch.equal(got, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


@pytest.mark.parametrize("n", [1, 4, 5, 8, 9, 64, 300, 2000])
@pytest.mark.parametrize("out,k", [(256, 512), (14336, 4096)])
def test_launches_of_products(ops, n, out, k):
    found, counted = kernels(product(ops, n, out, k)[0])
    assert found == counted and found in (1, 2)


@pytest.mark.parametrize("runs,nq", [([(1, 70)], 8), ([(1, 70)] * 256, 8), ([(1, 70)] * 257, 8), ([(2, 70)] * 1100, 8), ([(500, 700)], 16), ([(70, 70)] * 300, 16), ([(0, 70), (3, 3)], 8)])
def test_launches_of_attention(ops, runs, nq):
    found, counted = kernels(attention(ops, runs, nq)[0])
    assert found == counted


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 500), (128, 500)])
def test_launches_of_the_others(ops, rows, n):
    x = torch.zeros(n, 256, device="cuda")
    codes, scales = torch.empty(n, 256, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(2, -(-n // rows), device="cuda")
    found, counted = kernels(lambda: ops.quantize8(codes, scales, x, rows))
    assert found == counted == 1
    c = make([(3, 100), (1, 5)], 4, 2, 64)
    d = {key: t.cuda() for key, t in c.items()}
    new = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    found, counted = kernels(lambda: ops.cache_write8(d["k"], d["v"], d["ks"], d["vs"], new, new, d["table"], d["seq_slots"], d["cu"], d["lens"], 3))
    assert found == counted == 1


@pytest.mark.parametrize("runs,nq,longest", [([(1, 500), (2, 700), (1, 300)], 8, None), ([(200, 500), (300, 700), (100, 300)], 16, 700)])
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1, 10 ** 6])
def test_pages_that_do_not_exist(ops, runs, nq, longest, bad):
    """A sequence whose table names none gets something; nothing else is read or written, and the others get what they should."""
    dim, nkv, new = 64, 2, max(t for t, _ in runs)
    c = make(runs, nq, nkv, dim, seed=11)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    c["table"][c["seq_slots"][1], 3] = bad
    c["table"][c["seq_slots"][1], 9] = bad
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.full((c["q"].shape[0] + 1, nq * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention8(out[:-1], d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], dim ** -0.5, nq, nkv, dim, PAGE, new, max_len=longest)
    off = (out[:-1].cpu().to(F64) - want).abs()
    first, end = int(c["cu"][1]), int(c["cu"][2])
    right = (off <= bound).all(-1)
    assert bool(right[:first].all()) and bool(right[end:].all()) and bool((out[-1] == 7).all())
    ops.check_status()


@pytest.mark.parametrize("new", [1, 4, 200])
def test_writing_and_reading_in_turn_on_another_stream(ops, new):
    """Rows go into the cache and are read in the same step, step after step, without a wait of the host; then the same steps captured."""
    nq, nkv, dim, steps = 8, 2, 64, 6
    seqs, longest = 3, 64 + new * steps
    pages = -(-longest // PAGE)
    g = torch.Generator().manual_seed(new)
    table = torch.randperm(seqs * pages, generator=g).to(torch.int32).view(seqs, pages).cuda()
    slots, cu = torch.arange(seqs, dtype=torch.int32).cuda(), (torch.arange(seqs + 1) * new).to(torch.int32).cuda()
    lens = [torch.tensor([new * (i + 1)] * seqs, dtype=torch.int32).cuda() for i in range(steps)]
    k, v = (torch.randn(steps, seqs * new, nkv, dim, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(steps, seqs * new, nq, dim, generator=g).bfloat16().cuda()

    def run(pools, out):
        kc, vc, ks, vs = pools
        for i in range(steps):
            ops.cache_write8(kc, vc, ks, vs, k[i], v[i], table, slots, cu, lens[i], new)
            ops.attention8(out[i], q[i], kc, vc, ks, vs, table, slots, cu, lens[i], dim ** -0.5, nq, nkv, dim, PAGE, new)

    def fresh():
        kc, vc = (torch.full((seqs * pages, nkv, PAGE, dim), 0x7F, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        return kc, vc, torch.full((seqs * pages, nkv), 3.0, device="cuda"), torch.full((seqs * pages, nkv), 3.0, device="cuda")

    results = []
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        pools, out = fresh(), torch.empty(steps, seqs * new, nq * dim, dtype=torch.bfloat16, device="cuda")
        run(pools, out)
        results.append(out)
        again, out = fresh(), torch.empty_like(out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run(again, out)
        for _ in range(2):                                    # the second time over its own pages: each is written from its first position on
            graph.replay()
        results.append(out)
    torch.cuda.synchronize()
    assert torch.equal(results[0], results[1])
    # The last step against the definition, over the codes that stand now.
    c = dict(q=q[-1].cpu(), k=pools[0].cpu(), v=pools[1].cpu(), ks=pools[2].cpu(), vs=pools[3].cpu(), table=table.cpu(), seq_slots=slots.cpu(), cu=cu.cpu(), lens=lens[-1].cpu())
    want, bound = reference(c, dim ** -0.5, 0, 8)
    off = (results[0][-1].cpu().to(F64) - want).abs()
    assert bool((off <= bound).all())


@pytest.mark.parametrize("n", [1, 8, 20, 300])
def test_products_beyond_32_bits(ops, n):
    """More than 2^31 codes: first and last rows against 64 bits."""
    out, k = 140000, 16384
    codes = torch.randint(0, 120, (out, k), dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.exp2(torch.randint(-9, -6, (k // 128, -(-out // 128)), device="cuda").float())
    x, y = torch.randn(n, k, device="cuda").bfloat16(), torch.empty(n, out, dtype=torch.bfloat16, device="cuda")
    made, x_scales = torch.empty(n, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(k // 128, n, device="cuda")
    ops.quantize8(made, x_scales, x, 1)
    ops.linear8(y, x, codes, scales)
    wide = made.float().double() * x_scales.t().double().repeat_interleave(128, 1)
    for rows in (slice(0, 64), slice(out - 64, out)):
        w = codes[rows].float().double() * scales.t()[torch.arange(out, device="cuda")[rows] // 128].double().repeat_interleave(128, 1)
        want = wide @ w.t()
        # a 32-bit sum of 16,384 products, off by at most 2^-23 a step of their sizes, and one rounding to bfloat16
        bound = wide.abs() @ w.abs().t() * 16384 * 2.0 ** -23 + want.abs() * 2.0 ** -8
        assert bool(((y[:, rows].double() - want).abs() <= bound).all())


def test_quantising_beyond_32_bits(ops):
    n, k = 70000, 32768
    x = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_()
    codes = torch.empty(n, k, dtype=torch.uint8, device="cuda").view(E4M3)
    for rows in (1, 128):
        scales = torch.empty(k // 128, -(-n // rows), device="cuda")
        ops.quantize8(codes, scales, x, rows)
        few, some = torch.empty(112, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(k // 128, -(-112 // rows), device="cuda")
        ops.quantize8(few, some, x[-112:], rows)              # 70,000 = 546 x 128 + 112
        assert torch.equal(codes[-112:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scales[:, -some.shape[1]:], some)


def test_a_cache_beyond_32_bits(ops):
    """Pools of more than 2^32 bytes: a sequence whose pages are the first and the last ones."""
    nq, nkv, dim, length = 16, 8, 128, 200
    pages = 2 ** 32 // (nkv * PAGE * dim) + 50
    pools = [torch.zeros(pages, nkv, PAGE, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)]
    scales = [torch.ones(pages, nkv, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(length, nkv, dim, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(length, nq, dim, generator=g).bfloat16()
    small = [torch.zeros(4, nkv, PAGE, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)], [torch.ones(4, nkv, device="cuda") for _ in range(2)]
    outs = []
    for (kc, vc), (ks, vs), order in ((pools, scales, [pages - 1, 0, pages - 2, 1]), (*small, [0, 1, 2, 3])):
        table, slots = torch.tensor([order], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
        for new in (1, length):
            cu, lens = torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([length], dtype=torch.int32).cuda()
            out = torch.empty(new, nq * dim, dtype=torch.bfloat16, device="cuda")
            if new == length:
                ops.cache_write8(kc, vc, ks, vs, k.cuda(), v.cuda(), table, slots, cu, lens, new)
            ops.attention8(out, q[-new:].cuda(), kc, vc, ks, vs, table, slots, cu, lens, dim ** -0.5, nq, nkv, dim, PAGE, new)
            outs.append(out.cpu())
        cu = torch.tensor([0, 1], dtype=torch.int32).cuda()
        out = torch.empty(1, nq * dim, dtype=torch.bfloat16, device="cuda")
        ops.attention8(out, q[-1:].cuda(), kc, vc, ks, vs, table, slots, cu, lens, dim ** -0.5, nq, nkv, dim, PAGE, 1)
        outs.append(out.cpu())
    assert bool(outs[1].abs().max() > 0) and all(torch.equal(a, b) for a, b in zip(outs[:3], outs[3:]))


def test_long_runs_in_turns(ops):
    """Pages are widened for as many sequences at once as half a gigabyte holds: six with room for 32,768 positions each come in two turns."""
    nq, nkv, dim, longest = 32, 8, 128, 32768
    runs = [(100, 200), (0, 50), (7, 7), (100, 1000), (64, 640), (33, 90)]
    c = make(runs, nq, nkv, dim, seed=21)
    want, bound = reference(c, dim ** -0.5, 0, 8)
    c["table"] = torch.cat([c["table"], torch.full((c["table"].shape[0], longest // PAGE - c["table"].shape[1]), -1, dtype=torch.int32)], 1)
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.full((c["q"].shape[0] + 1, nq * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.lib().ti_attention8_widens(6, 100, nq, nkv, dim, longest) == 1
    assert ops.attention8_workspace(6, 100, nq, nkv, dim, longest) <= 2 ** 29 + 2 ** 20
    found, counted = kernels(lambda: ops.attention8(out[:-1], d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], dim ** -0.5, nq, nkv, dim,
                                                    PAGE, 100))
    torch.cuda.synchronize()
    assert found == counted == 4
    assert bool(((out[:-1].cpu().to(F64) - want).abs() <= bound).all()) and bool((out[-1] == 7).all())
    ops.check_status()


def test_lengths_beyond_the_table(ops):
    """A length that the table's row has no pages for: what lies beyond reads as zeros, the others get what they should."""
    runs, nq, nkv, dim = [(2, 300), (2, 500), (1, 70)], 8, 2, 64
    c = make(runs, nq, nkv, dim, seed=2)
    want, bound = reference(c, dim ** -0.5, 0, 11)
    c["lens"][1] = 64 * (c["table"].shape[1] + 40)
    c["table"] = c["table"][:int(c["seq_slots"].max()) + 1].contiguous()
    d = {key: t.cuda() for key, t in c.items()}
    out = torch.empty(c["q"].shape[0], nq * dim, dtype=torch.bfloat16, device="cuda")
    ops.attention8(out, d["q"], d["k"], d["v"], d["ks"], d["vs"], d["table"], d["seq_slots"], d["cu"], d["lens"], dim ** -0.5, nq, nkv, dim, PAGE, 2)
    right = ((out.cpu().to(F64) - want).abs() <= bound).all(-1)
    assert bool(right[:2].all()) and bool(right[4:].all())
    ops.check_status()


@pytest.mark.parametrize("n", [4, 20, 33, 64, 1000])
@pytest.mark.parametrize("name", ["EPI_NONE", "EPI_XIELU", "EPI_GELU_ERF", "EPI_GELU_TANH", "EPI_RELU2", "EPI_F32_OUT"])
def test_launches_with_an_activation(ops, n, name):
    """An activation that is a launch of its own is counted, and gives what it gives over strided rows, where it is none."""
    out, k, epilogue = 1040, 512, getattr(ops, name)
    g = torch.Generator().manual_seed(n)
    w, x = torch.randn(out, k, generator=g).bfloat16().cuda(), torch.randn(n, k, generator=g).bfloat16().cuda()
    codes, scales = torch.empty(out, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(4, -(-out // 128), device="cuda")
    ops.quantize8(codes, scales, w, 128)
    dtype = torch.float32 if name == "EPI_F32_OUT" else torch.bfloat16
    dense, wide = torch.empty(n, out, dtype=dtype, device="cuda"), torch.full((n, out + 16), 7.0, dtype=dtype, device="cuda")
    act = (0.8, 0.8, 0.5, -1e-6)
    found, counted = kernels(lambda: ops.linear8(dense, x, codes, scales, None, epilogue, act))
    assert found == counted
    found, counted = kernels(lambda: ops.linear8(wide[:, :out], x, codes, scales, None, epilogue, act))
    assert found == counted and torch.equal(dense, wide[:, :out]) and bool((wide[:, out:] == 7).all())


@pytest.mark.parametrize("act", [(0.75, 0.875, 0.5, -1e-6), (0.8, 0.8, 0.5, -1e-6)])
@pytest.mark.parametrize("n,out", [(33, 1040), (64, 333), (700, 4096), (1, 64)])
def test_xielu_is_the_library_s_own(ops, n, out, act):
    """Factors that are bfloat16 numbers, and others: the bits of the sums' own activation."""
    g = torch.Generator().manual_seed(n)
    w, x = torch.randn(out, 512, generator=g).bfloat16().cuda(), torch.randn(n, 512, generator=g).bfloat16().cuda()
    codes, scales = torch.empty(out, 512, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(4, -(-out // 128), device="cuda")
    ops.quantize8(codes, scales, w, 128)
    plain, got, want = (torch.empty(n, out, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    ops.linear8(plain, x, codes, scales)
    ops.linear8(got, x, codes, scales, None, ops.EPI_XIELU, act)
    ops.xielu(want, plain, *act)
    assert torch.equal(got, want)
