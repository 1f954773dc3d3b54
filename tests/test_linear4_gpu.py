"""Products with weights of 4 bits against the definition in 64 bits.

Bounds: a sum of m 32-bit additions in any tree with a longest path of d additions is off by at most d 2^-23 times the sum of the magnitudes (2^-23:
tensor cores may cut instead of round), and a rounding to bfloat16 adds 2^-8 of the result (half its widest step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def pack(code):
    """codes [out, k] -> words [out, k / 8]: even k in the low half, odd k in the high half, ascending."""
    c = code.long().view(code.shape[0], -1, 8)
    word = sum(c[:, :, i] << (4 * (i // 2) + 16 * (i % 2)) for i in range(8))
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def case(n, out, k, group, dtype, with_zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 16, (out, k), generator=g)
    scales = ((torch.rand(k // group, out, generator=g) + 0.5) * 0.01).to(dtype)
    zeros = torch.randint(0, 16, (k // group, out), generator=g).to(torch.uint8) if with_zeros else None
    x = torch.randn(n, k, generator=g).to(dtype)
    z = zeros.t().repeat_interleave(group, 1).to(F64) if with_zeros else 8.0
    w = (code.to(F64) - z) * scales.t().to(F64).repeat_interleave(group, 1)
    return code, scales, zeros, x, w


def bounds(x, w, dtype, group):
    want = x.to(F64) @ w.t()
    total = x.to(F64).abs() @ w.t().abs()
    k = x.shape[1]
    if dtype == torch.float32:
        return want, total * (40 + k / 1024) * 2.0 ** -23
    return want, total * (group + k / group + 16) * 2.0 ** -23 + want.abs() * 2.0 ** -8


def check(ops, n, out, k, group, dtype, with_zeros, seed=0):
    code, scales, zeros, x, w = case(n, out, k, group, dtype, with_zeros, seed)
    y = torch.full((n, out), float("nan"), dtype=dtype, device="cuda")
    ops.linear4(y, x.cuda(), pack(code).cuda(), scales.cuda(), zeros.cuda() if with_zeros else None)
    want, bound = bounds(x, w, dtype, group)
    off = (y.cpu().to(F64) - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,out,groups", [(1, 1, 1), (1, 320, 3), (5, 333, 5), (8, 640, 7), (9, 100, 2), (16, 1203, 9), (17, 257, 3), (33, 512, 4),
                                          (64, 130, 6), (65, 48, 5), (130, 7, 1), (300, 129, 2)])
def test_sizes(ops, dtype, group, n, out, groups):
    check(ops, n, out, group * groups, group, dtype, (out + groups) % 2 == 0, seed=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,out,k,group,with_zeros", [(1, 6144, 4096, 128, True), (3, 4096, 21504, 64, False), (12, 2051, 8192, 128, True),
                                                      (2, 50257, 512, 32, True), (40, 4096, 4096, 128, False), (64, 3001, 2048, 32, True), (5, 2051, 8192, 32, True),
                                                      (1, 2600, 8320, 64, True), (8, 2048, 9216, 128, False)])
def test_layer_sizes(ops, dtype, n, out, k, group, with_zeros):
    check(ops, n, out, k, group, dtype, with_zeros)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [0, 2, 20, 70])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strided_rows(ops, dtype, n, shift):
    code, scales, zeros, x, w = case(n, 95, 192, 64, dtype, True, 3)
    wide = torch.zeros(n + 1, 192 + 40 + shift, dtype=dtype, device="cuda")
    xs = wide[:n, shift:shift + 192]
    xs.copy_(x)
    held = torch.zeros(n + 1, 131, dtype=dtype, device="cuda")
    ops.linear4(held[:n, 3:98], xs, pack(code).cuda(), scales.cuda(), zeros.cuda())
    want, bound = bounds(x, w, dtype, 64)
    assert bool(((held[:n, 3:98].cpu().to(F64) - want).abs() <= bound).all())
    assert not held[:, :3].any() and not held[:, 98:].any() and not held[n:].any()      # nothing beside the rows


@pytest.mark.parametrize("out", [96, 95])
def test_unaligned_scales(ops, out):
    """Scales and zeros from an address that takes no wide reads."""
    code, scales, zeros, x, w = case(4, out, 256, 32, torch.bfloat16, True, 5)
    s = torch.zeros(scales.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(scales)
    z = torch.zeros(zeros.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(zeros)
    s.copy_(scales); z.copy_(zeros)
    y = torch.empty(4, out, dtype=torch.bfloat16, device="cuda")
    ops.linear4(y, x.cuda(), pack(code).cuda(), s, z)
    want, bound = bounds(x, w, torch.bfloat16, 32)
    assert bool(((y.cpu().to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("n", [3, 30])
def test_unrounded_sums_and_activations(ops, n):
    code, scales, zeros, x, w = case(n, 77, 256, 64, torch.bfloat16, False, 7)
    args = (x.cuda(), pack(code).cuda(), scales.cuda())
    y = torch.empty(n, 77, dtype=torch.float32, device="cuda")
    ops.linear4(y, *args, epilogue=ops.EPI_F32_OUT)
    want = x.to(F64) @ w.t()
    assert bool(((y.cpu().to(F64) - want).abs() <= (x.to(F64).abs() @ w.t().abs()) * 90 * 2.0 ** -23).all())
    plain = torch.empty(n, 77, dtype=torch.bfloat16, device="cuda")
    ops.linear4(plain, *args)
    assert torch.equal(plain, y.to(torch.bfloat16))                                      # the same sums, rounded
    act = (0.8, 0.9, 0.5, -1e-6)
    got, want_act = torch.empty_like(plain), torch.empty_like(plain)
    ops.linear4(got, *args, epilogue=ops.EPI_XIELU, act=act)
    ops.xielu(want_act, plain, *act)
    assert torch.equal(got, want_act)


def test_infinities_stay_in_their_rows(ops):
    code, scales, zeros, x, w = case(6, 40, 128, 32, torch.bfloat16, False, 9)
    x[2, 5], x[4, 7] = float("inf"), float("nan")
    y = torch.empty(6, 40, dtype=torch.bfloat16, device="cuda")
    ops.linear4(y, x.cuda(), pack(code).cuda(), scales.cuda())
    y = y.cpu()
    rows = [0, 1, 3, 5]
    want, bound = bounds(x[rows], w, torch.bfloat16, 32)
    assert bool(((y[rows].to(F64) - want).abs() <= bound).all())
    assert not torch.isfinite(y[2]).any() and bool(torch.isnan(y[4]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_token_does_not_depend_on_its_step(ops, dtype):
    """32-bit: bit for bit. bfloat16: the same up to one rounding."""
    code, scales, zeros, x, w = case(40, 200, 1024, 128, dtype, True, 11)
    args = (pack(code).cuda(), scales.cuda(), zeros.cuda())
    whole = torch.empty(40, 200, dtype=dtype, device="cuda")
    ops.linear4(whole, x.cuda(), *args)
    for a, b in ((0, 1), (1, 9), (9, 40)):
        part = torch.empty(b - a, 200, dtype=dtype, device="cuda")
        ops.linear4(part, x[a:b].cuda(), *args)
        if dtype == torch.float32:
            assert torch.equal(part, whole[a:b])
        else:
            want, bound = bounds(x[a:b], w, dtype, 128)
            assert bool(((part.cpu().to(F64) - want).abs() <= bound).all())


def test_other_stream_and_graph(ops):
    code, scales, zeros, x, w = case(4, 300, 512, 64, torch.bfloat16, False, 13)
    dev = [t.cuda() for t in (x, pack(code), scales)]
    want = torch.empty(4, 300, dtype=torch.bfloat16, device="cuda")
    ops.linear4(want, *dev)
    got = torch.zeros_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear4(got, *dev)
    side.synchronize()
    assert torch.equal(got, want)
    replayed = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear4(replayed, *dev)
    dev[0].neg_()
    graph.replay()
    assert torch.equal(replayed, -want)


# ------------------------------------------------------------------------------ the codes of a matrix
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("with_zeros", [False, True])
def test_quantize(ops, dtype, group, with_zeros):
    """Codes, scales and zeros by the rule, each step rounded as written, and no weight further off than half a step (and the rounding of the scale)."""
    torch.manual_seed(1)
    out, k = 37, 5 * group
    w = (torch.randn(out, k) * 0.02).to(dtype)
    w[3] = 0.0
    w[4, :group] = w[4, :group].abs()
    w[5, group:2 * group] = 0.25
    codes = torch.empty(out, k // 8, dtype=torch.int32, device="cuda")
    scales = torch.empty(5, out, dtype=dtype, device="cuda")
    zeros = torch.empty(5, out, dtype=torch.uint8, device="cuda") if with_zeros else None
    ops.quantize4(codes, scales, w.cuda(), zeros)
    grouped = w.float().view(out, 5, group)
    top, low = grouped.amax(2).clamp_min(0), grouped.amin(2).clamp_max(0)
    scale = (((top - low) / 15.0) if with_zeros else (torch.maximum(top, -low) / 7.0)).to(dtype).float()
    safe = torch.where(scale > 0, scale, 1.0)
    zero = torch.where(scale > 0, torch.round(-low / safe).clamp_max(15), 0.0) if with_zeros else torch.full_like(scale, 8.0)
    code = (zero[:, :, None] + torch.where(scale[:, :, None] > 0, torch.round(grouped / safe[:, :, None]), 0.0)).clamp(0 if with_zeros else 1, 15)
    assert torch.equal(scales.cpu().float(), scale.t())
    if with_zeros:
        assert torch.equal(zeros.cpu().float(), zero.t())
    assert torch.equal(codes.cpu(), pack(code.reshape(out, k)))
    back = (code - zero[:, :, None]) * scale[:, :, None]
    assert bool(((back - grouped).abs() <= scale[:, :, None] * (0.5 + (1.0 if with_zeros else 0.0) * 0.5 + 15 * 2.0 ** -8) + 1e-12).all())


def test_quantize_then_product_on_one_stream(ops):
    """The product right behind the kernel that makes its codes."""
    torch.manual_seed(2)
    w = torch.randn(512, 1024).to(torch.bfloat16).cuda()
    x = torch.randn(3, 1024).to(torch.bfloat16).cuda()
    codes, scales = torch.zeros(512, 128, dtype=torch.int32, device="cuda"), torch.zeros(8, 512, dtype=torch.bfloat16, device="cuda")
    ops.quantize4(codes, scales, w)
    want = torch.empty(3, 512, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ops.linear4(want, x, codes, scales)
    for _ in range(20):
        codes.zero_()
        got = torch.empty_like(want)
        ops.quantize4(codes, scales, w)
        ops.linear4(got, x, codes, scales)
        assert torch.equal(got, want)


def test_refusals(ops):
    y, x = torch.empty(2, 64, device="cuda"), torch.empty(2, 128, device="cuda")
    codes, scales = torch.zeros(64, 16, dtype=torch.int32, device="cuda"), torch.ones(2, 64, device="cuda")
    ops.linear4(y, x, codes, scales)
    bad = [dict(x=x.half()), dict(x=x.cpu()), dict(y=y.bfloat16()), dict(y=y[:1]), dict(codes=codes.long()), dict(codes=codes[:, :8]),
           dict(codes=codes.t().contiguous().t()), dict(scales=scales.bfloat16()), dict(scales=torch.ones(8, 64, device="cuda")),
           dict(scales=torch.ones(3, 64, device="cuda")), dict(zeros=torch.zeros(2, 64, dtype=torch.int32, device="cuda")),
           dict(zeros=torch.zeros(2, 63, dtype=torch.uint8, device="cuda")), dict(x=torch.empty(128, 2, device="cuda").t()), dict(epilogue=99),
           dict(codes=torch.zeros(64 * 16 + 1, dtype=torch.int32, device="cuda")[1:].view(64, 16)), dict(x=x[0]),
           dict(epilogue=ops.EPI_F32_OUT, x=x.bfloat16(), scales=scales.bfloat16(), y=y.bfloat16())]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.linear4(**{**dict(y=y, x=x, codes=codes, scales=scales), **change})
    for change in (dict(w=x.half()), dict(codes=codes[:, :8]), dict(scales=torch.ones(8, 64, device="cuda")),
                   dict(zeros=torch.zeros(1, 64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ops.KernelError):
            ops.quantize4(**{**dict(codes=codes, scales=scales, w=torch.zeros(64, 128, device="cuda")), **change})
