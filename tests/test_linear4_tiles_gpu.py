"""Products with weights of 4 bits at sizes where tiles of 256 rows are more than the GPU's blocks, and every tile is one block's or cut between two.

Bounds as for the other sizes: a sum of m 32-bit additions with a longest path of d is off by at most d 2^-23 times the sum of the magnitudes, and a rounding to
bfloat16 adds 2^-8 of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def case(n, out, k, group, with_zeros, seed):
    """x, codes, scales and zeros on the device, and W in 64 bits there."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = torch.randint(0, 16, (out, k), generator=g, device="cuda")
    scales = ((torch.rand(k // group, out, generator=g, device="cuda") + 0.5) * 0.01).to(torch.bfloat16)
    zeros = torch.randint(0, 16, (k // group, out), generator=g, device="cuda").to(torch.uint8) if with_zeros else None
    x = torch.randn(n, k, generator=g, device="cuda").to(torch.bfloat16)
    words = sum(code.view(out, -1, 8)[:, :, i] << (4 * (i // 2) + 16 * (i % 2)) for i in range(8))
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    z = zeros.t().repeat_interleave(group, 1).to(F64) if with_zeros else 8.0
    return x, words, scales, zeros, (code.to(F64) - z) * scales.t().to(F64).repeat_interleave(group, 1)


@pytest.mark.parametrize("n", [9, 16, 40, 100])
@pytest.mark.parametrize("out,k,group,with_zeros", [(40001, 640, 128, False), (38400, 576, 64, True), (41000, 96, 32, True), (20000, 1280, 32, False)])
def test_more_tiles_than_blocks(ops, n, out, k, group, with_zeros):
    x, words, scales, zeros, w = case(n, out, k, group, with_zeros, out + n)
    y = torch.full((n, out), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.linear4(y, x, words, scales, zeros)
    want, total = x.to(F64) @ w.t(), x.to(F64).abs() @ w.t().abs()
    bound = total * (group + k / group + 16) * 2.0 ** -23 + want.abs() * 2.0 ** -8
    assert bool(((y.to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("n,out,k", [(20, 9000, 256), (33, 4099, 1024), (9, 40001, 640), (8, 3000, 8192)])
def test_results_leave_alike(ops, n, out, k):
    """The same sums unrounded, rounded and through the activations, from tiles that are whole and from joined ones."""
    x, words, scales, zeros, w = case(n, out, k, 128, True, 3)
    sums = torch.full((n, out), float("nan"), dtype=torch.float32, device="cuda")
    ops.linear4(sums, x, words, scales, zeros, epilogue=ops.EPI_F32_OUT)
    want, total = x.to(F64) @ w.t(), x.to(F64).abs() @ w.t().abs()
    assert bool(((sums.to(F64) - want).abs() <= total * (128 + k / 128 + 16) * 2.0 ** -23).all())
    held = torch.zeros(n + 1, out + 5, dtype=torch.bfloat16, device="cuda")
    ops.linear4(held[:n, 3:out + 3], x, words, scales, zeros)
    plain = held[:n, 3:out + 3].contiguous()
    assert torch.equal(plain, sums.to(torch.bfloat16))
    assert not held[:, :3].any() and not held[:, out + 3:].any() and not held[n:].any()
    act = (0.8, 0.9, 0.5, -1e-6)
    got, want_act = torch.empty_like(plain), torch.empty_like(plain)
    ops.linear4(got, x, words, scales, zeros, epilogue=ops.EPI_XIELU, act=act)
    ops.xielu(want_act, plain, *act)
    assert torch.equal(got, want_act)
