"""The same bits from the same product, many times over, where a block goes through its ring of stages again and again."""
import pytest
import torch

from test_linear4_tiles_gpu import case

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.mark.parametrize("n,out,k,group,with_zeros", [(8, 65536, 4096, 128, False), (16, 32768, 8192, 32, True), (40, 28672, 8192, 64, True), (4, 8192, 28672, 128, True)])
def test_the_same_bits(n, out, k, group, with_zeros):
    from tileinfer_b200.kernels import ops
    x, words, scales, zeros, w = case(n, out, k, group, with_zeros, 5)
    ys = [torch.empty(n, out, dtype=torch.bfloat16, device="cuda") for _ in range(10)]
    for _ in range(10):
        for y in ys:
            ops.linear4(y, x, words, scales, zeros)
        assert all(torch.equal(y, ys[0]) for y in ys[1:])
    ops.check_status()
    want, total = x.to(F64) @ w.t(), x.to(F64).abs() @ w.t().abs()
    bound = total * (group + k / group + 16) * 2.0 ** -23 + want.abs() * 2.0 ** -8
    assert bool(((ys[0].to(F64) - want).abs() <= bound).all())
