"""Products of e4m3 codes against the definition in 64 bits.

Bound of a result y = sum_g sx sw part_g: a part's at most 128 products are exact and added in 32 bits with at most 128 roundings (2^-23 of the sum of sizes each,
cut off or rounded), its scale's product is rounded (2^-23), and the groups' sum takes a rounding a group: |y'| <= (130 + groups) 2^-23 sum |x w|; one more
rounding to bfloat16 is 2^-8 |y|."""
import pytest
import torch

from numbers8 import BLOCK, E4M3, F64, blocks

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -23


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def weights(out, k, seed=0, any_scale=False):
    """Codes of every finite kind; scales around those of trained weights, powers of two or not."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = (torch.randn(out, k, device="cuda", generator=g) * 100).clamp_(-448, 448).to(E4M3)
    scales = torch.rand(-(-k // BLOCK), -(-out // BLOCK), device="cuda", generator=g) + 0.5
    return codes, scales * 2.0 ** -12 if any_scale else torch.exp2(torch.floor(4 * scales) - 14)


def inputs(n, k, seed=0, given=False, any_scale=False):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    x = torch.randn(n, k, device="cuda", generator=g) * torch.exp(torch.randn(n, 1, device="cuda", generator=g))
    if not given:
        return x.to(torch.bfloat16), None
    scales = torch.rand(-(-k // BLOCK), n, device="cuda", generator=g) + 0.5
    return (x * 60).clamp_(-448, 448).to(E4M3), scales / 50 if any_scale else torch.exp2(torch.floor(4 * scales) - 8)


def widened(codes, scales, rows):
    n, k = codes.shape
    return codes.to(F64) * scales.to(F64).t().repeat_interleave(rows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def reference(x, x_scales, codes, scales):
    """(result, bound of the 32-bit sums), on the device in 64 bits."""
    if x_scales is None:
        v, s = blocks(x.float().cpu(), 1)
        x, x_scales = v.cuda(), s.cuda()
    a, w = widened(x, x_scales, 1), widened(codes, scales, BLOCK)
    return a @ w.t(), a.abs() @ w.abs().t() * ((130 + x_scales.shape[0]) * EPS)


def check(ops, n, out, k, given=False, f32=False, seed=0, any_scale=False):
    codes, scales = weights(out, k, seed, any_scale)
    x, x_scales = inputs(n, k, seed, given, any_scale)
    y = torch.full((n + 1, out), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    ops.linear8(y[:n], x, codes, scales, x_scales, ops.EPI_F32_OUT if f32 else ops.EPI_NONE)
    want, bound = reference(x, x_scales, codes, scales)
    if not f32:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    off = (y[:n].to(F64) - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
    assert bool((y[n:] == 7).all())
    ops.check_status()


SIZES = [(1, 1, 16), (1, 128, 128), (1, 300, 2064), (5, 320, 96), (3, 129, 144), (8, 256, 4096), (9, 1000, 1040), (16, 2048, 512), (17, 513, 384), (32, 640, 272),
         (33, 140, 4112), (64, 4096, 1024), (65, 384, 256), (100, 130, 640), (128, 1024, 1024), (129, 264, 272), (200, 5000, 528), (256, 512, 128), (300, 777, 2000),
         (511, 1536, 144), (1000, 520, 16), (2048, 300, 384), (2050, 1280, 1168)]


@pytest.mark.parametrize("n,out,k", SIZES)
@pytest.mark.parametrize("given", [False, True])
def test_sizes(ops, n, out, k, given):
    check(ops, n, out, k, given, seed=n + out + k)


@pytest.mark.parametrize("n,out,k", [(1, 21504, 4096), (16, 4096, 21504), (64, 6144, 4096), (256, 4096, 4096), (700, 4096, 2048), (2048, 4096, 4096)])
@pytest.mark.parametrize("given", [False, True])
def test_sizes_of_real_layers(ops, n, out, k, given):
    check(ops, n, out, k, given, any_scale=True)


@pytest.mark.parametrize("n,out,k", [(1, 5000, 512), (7, 300, 4096), (40, 333, 640), (130, 1000, 272), (600, 1024, 640), (1500, 1000, 1024)])
def test_sums_in_32_bits(ops, n, out, k):
    for given in (False, True):
        check(ops, n, out, k, given, f32=True, any_scale=given)


@pytest.mark.parametrize("n,out", [(3, 200), (40, 513), (300, 1024), (1200, 2000)])
@pytest.mark.parametrize("epilogue", ["xielu", "gelu_erf", "gelu_tanh", "relu2"])
def test_epilogues(ops, n, out, epilogue):
    """Applied to the rounded sum, as the framework's other products do it: the same bits as on a result that was rounded first."""
    codes, scales = weights(out, 400)
    x, _ = inputs(n, 400)
    plain, y = (torch.empty(n, out, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.linear8(plain, x, codes, scales)
    act = (0.8, 0.8, 0.5, -1e-6)
    ops.linear8(y, x, codes, scales, None, {"xielu": ops.EPI_XIELU, "gelu_erf": ops.EPI_GELU_ERF, "gelu_tanh": ops.EPI_GELU_TANH, "relu2": ops.EPI_RELU2}[epilogue], act)
    want = torch.empty_like(plain)
    if epilogue == "xielu":
        ops.xielu(want, plain, *act)
    elif epilogue == "relu2":
        want = (plain.float().clamp_min(0) ** 2).to(torch.bfloat16)
    else:
        ops.gelu(want, plain, ops.ACT_GELU_ERF if epilogue == "gelu_erf" else ops.ACT_GELU_TANH)
    assert torch.equal(y, want)


@pytest.mark.parametrize("n", [1, 12, 70, 400])
@pytest.mark.parametrize("x_pitch,x_first", [(512, 0), (392, 0), (393, 1), (385, 0)])
def test_rows_of_any_pitch(ops, n, x_pitch, x_first):
    codes, scales = weights(200, 384)
    wide = torch.randn(n, x_pitch, device="cuda").to(torch.bfloat16)
    x = wide[:, x_first:x_first + 384]
    y, apart = torch.empty(n, 200, dtype=torch.bfloat16, device="cuda"), torch.full((n, 333), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.linear8(y, x.contiguous(), codes, scales)
    ops.linear8(apart[:, 5:205], x, codes, scales)
    assert torch.equal(apart[:, 5:205], y)
    assert bool((apart[:, :5] == 7).all()) and bool((apart[:, 205:] == 7).all())


@pytest.mark.parametrize("n", [1, 40, 300])
def test_one_row_for_all_tokens(ops, n):
    codes, scales = weights(200, 384)
    x = torch.randn(1, 384, device="cuda").to(torch.bfloat16)
    y, one = torch.empty(n, 200, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 200, dtype=torch.bfloat16, device="cuda")
    ops.linear8(y, x.expand(n, 384), codes, scales)
    want, bound = reference(x, None, codes, scales)
    assert bool(((y.to(F64) - want).abs() <= bound + (want.abs() + bound) * 2.0 ** -8).all())
    ops.linear8(one, x, codes, scales)


@pytest.mark.parametrize("n", [2, 70, 300, 1300])
def test_what_is_not_finite_stays_in_its_row_and_column(ops, n):
    codes, scales = weights(260, 272)
    x, _ = inputs(n, 272)
    clean = torch.empty(n, 260, dtype=torch.bfloat16, device="cuda")
    ops.linear8(clean, x, codes, scales)
    x[1, 200] = float("inf")
    codes.view(torch.uint8)[130, 7] = 0x7F
    y = torch.empty_like(clean)
    ops.linear8(y, x, codes, scales)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[:, 130]).all())
    rows, columns = [t for t in range(n) if t != 1], [o for o in range(260) if o != 130]
    assert torch.equal(y[rows][:, columns], clean[rows][:, columns])


@pytest.mark.parametrize("n,out,k,given", [(4, 2048, 4096, False), (100, 512, 4096, False), (1100, 1024, 512, False), (1100, 1024, 512, True)])
def test_graphs_streams_and_work_spaces(ops, n, out, k, given):
    """Captured twice, replayed in turn on two streams, with a caller's work space and without."""
    made = [(weights(out, k, s), inputs(n, k, s, given)) for s in (1, 2)]
    want = []
    for (codes, scales), (x, xs) in made:
        y = torch.empty(n, out, dtype=torch.bfloat16, device="cuda")
        ops.linear8(y, x, codes, scales, xs)
        want.append(y)
    need = ops.linear8_workspace(n, out, k, given)
    if need:
        y = torch.empty_like(want[0])
        ops.linear8(y, made[0][1][0], *made[0][0], made[0][1][1], workspace=torch.full((need,), 255, dtype=torch.uint8, device="cuda"))
        assert torch.equal(y, want[0])
        with pytest.raises(ops.KernelError, match="work space"):
            ops.linear8(y, made[0][1][0], *made[0][0], made[0][1][1], workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    graphs, ys = [], [torch.empty_like(w) for w in want]
    for ((codes, scales), (x, xs)), y in zip(made, ys):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.linear8(y, x, codes, scales, xs)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for y, w in zip(ys, want):
        assert torch.equal(y, w)


@pytest.mark.parametrize("n,out,k", [(16, 4096, 8192), (300, 1024, 1024), (2048, 2048, 1024)])
def test_the_same_bits_every_time(ops, n, out, k):
    codes, scales = weights(out, k)
    x, _ = inputs(n, k)
    y, first = torch.empty(n, out, dtype=torch.bfloat16, device="cuda"), torch.empty(n, out, dtype=torch.bfloat16, device="cuda")
    ops.linear8(first, x, codes, scales)
    for _ in range(50):
        y.fill_(7.0)
        ops.linear8(y, x, codes, scales)
        assert torch.equal(y, first)
    ops.check_status()


def test_no_tokens(ops):
    codes, scales = weights(128, 64)
    ops.linear8(torch.empty(0, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), codes, scales)


def test_refusals(ops):
    codes, scales = weights(384, 192)
    x, xs = inputs(3, 192, given=True)
    y = torch.empty(3, 384, dtype=torch.bfloat16, device="cuda")
    good = dict(y=y, x=x, codes=codes, scales=scales, x_scales=xs)
    ops.linear8(**good)
    b = x.to(torch.bfloat16)
    for change in (dict(x=b), dict(x_scales=None), dict(x=x.cpu()), dict(y=y.float()), dict(epilogue=ops.EPI_F32_OUT), dict(codes=codes.view(torch.uint8)),
                   dict(scales=scales[:1]), dict(scales=scales.t().contiguous()), dict(x_scales=xs.t().contiguous()), dict(x_scales=xs.double()), dict(y=y[:, :383]),
                   dict(x=b.float(), x_scales=None), dict(codes=codes[:, :176]), dict(x=x[0]), dict(y=y.t().contiguous().t()), dict(epilogue=9),
                   dict(x=torch.empty(3 * 192 + 8, dtype=torch.uint8, device="cuda")[8:].view(3, 192).view(E4M3)),
                   dict(codes=torch.empty(384 * 192 + 8, dtype=torch.uint8, device="cuda")[8:].view(384, 192).view(E4M3))):
        with pytest.raises(ops.KernelError):
            ops.linear8(**{**good, **change})
    thin = torch.ones(2, 24, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.KernelError):                     # k is no multiple of 16
        ops.linear8(y[:2], thin, codes[:, :24].contiguous(), scales[:1], None)
