"""Products with 4-bit weights whose zeros are the largest that they take, 128: code - zero is a whole number that bfloat16 holds exactly up to there."""
import pytest
import torch

from test_linear4_gpu import bounds, case, pack

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,out,k", [(3, 100, 512), (20, 600, 4096), (8, 300, 8192)])
@pytest.mark.parametrize("low", [0, 16, 127, 128])
def test_zeros_up_to_the_largest(ops, dtype, group, n, out, k, low):
    code, scales, _, x, _ = case(n, out, k, group, dtype, False, 3)
    zeros = torch.randint(low, 129, (k // group, out), generator=torch.Generator().manual_seed(low)).to(torch.uint8)
    w = (code.to(F64) - zeros.t().repeat_interleave(group, 1).to(F64)) * scales.t().to(F64).repeat_interleave(group, 1)
    y = torch.full((n, out), float("nan"), dtype=dtype, device="cuda")
    ops.linear4(y, x.cuda(), pack(code).cuda(), scales.cuda(), zeros.cuda())
    want, bound = bounds(x, w, dtype, group)
    assert bool(((y.cpu().to(F64) - want).abs() <= bound).all())
