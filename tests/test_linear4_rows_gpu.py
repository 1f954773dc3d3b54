"""Products with 4-bit weights whose token rows lie in unusual places: one row for all tokens, rows that overlap, a single row of any pitch."""
import pytest
import torch

from test_linear4_gpu import bounds, case, pack

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def views(x, n, k):
    """Token rows as views of one stretch of x's elements, by name."""
    return {"one row for all": x[:k].expand(n, k), "overlapping": x.as_strided((n, k), (8, 1)), "overlapping, odd": x.as_strided((n, k), (3, 1)),
            "half a row apart": x.as_strided((n, k), (k // 2, 1))}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,out,k", [(3, 77, 256), (16, 1030, 4096), (40, 333, 8192), (7, 700, 8192)])
@pytest.mark.parametrize("kind", ["one row for all", "overlapping", "overlapping, odd", "half a row apart"])
def test_rows_that_share_elements(ops, dtype, n, out, k, kind):
    code, scales, zeros, x, w = case(n, out, k, 128, dtype, True, 3)
    x = views(x.reshape(-1).cuda(), n, k)[kind]
    y = torch.full((n, out), float("nan"), dtype=dtype, device="cuda")
    ops.linear4(y, x, pack(code).cuda(), scales.cuda(), zeros.cuda())
    want, bound = bounds(x.cpu(), w, dtype, 128)
    assert bool(((y.cpu().to(F64) - want).abs() <= bound).all())


@pytest.mark.parametrize("pitch", [0, 1, 8, 4096, 4104, 1 << 40])
def test_one_row_of_any_pitch(ops, pitch):
    """A single row's pitch means nothing."""
    code, scales, zeros, x, w = case(1, 1030, 8192, 128, torch.bfloat16, False, 4)
    row = x.reshape(-1).cuda().as_strided((1, 8192), (pitch, 1))
    y = torch.zeros(1, 1030, dtype=torch.bfloat16, device="cuda")
    ops.linear4(y, row, pack(code).cuda(), scales.cuda())
    want, bound = bounds(x, w, torch.bfloat16, 128)
    assert bool(((y.cpu().to(F64) - want).abs() <= bound).all())
