"""Codes of e4m3 and their scales: equal to the definition's, bit for bit."""
import pytest
import torch

from numbers8 import E4M3, blocks, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def run(ops, x, rows):
    n, k = x.shape
    codes = torch.full((n + 2, k), 0x55, dtype=torch.uint8, device="cuda").view(E4M3)          # two rows behind the last
    scales = torch.full((-(-k // 128), -(-n // rows)), -1.0, device="cuda")
    ops.quantize8(codes[:n], scales, x, rows)
    assert bool((codes[n:].view(torch.uint8) == 0x55).all())
    return codes[:n].float().cpu(), scales.cpu()


def check(ops, x, rows):
    codes, scales = run(ops, x.cuda(), rows)
    want, s = blocks(x, rows)
    assert torch.equal(scales.double(), s)
    assert same(codes, want)


def values(n, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, k, generator=g) * torch.exp(3 * torch.randn(n, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("n,k", [(1, 16), (1, 128), (3, 144), (16, 512), (17, 528), (127, 96), (128, 1040), (129, 640), (300, 2064)])
def test_sizes(ops, n, k, rows, dtype):
    check(ops, values(n, k, dtype, n + k), rows)


@pytest.mark.parametrize("rows", [1, 128])
def test_values_at_the_borders(ops, rows):
    """Ties, the largest of a scale and one step above, zeros, the smallest and largest numbers, what is not finite."""
    x = torch.zeros(13, 128)
    x[0] = torch.arange(128) / 64.0 + 1.0
    x[1, 0], x[2, 0], x[3, 0] = 448.0, 448.0 * (1 + 2.0 ** -23), 447.9
    x[4] = 448.0 * 2.0 ** torch.arange(0, -128, -1).float()
    x[5], x[6] = 2.0 ** -140, -2.0 ** -100
    x[7] = 3.4e38
    x[8, :3] = torch.tensor([float("inf"), float("nan"), -float("inf")])
    x[9] = float("inf")
    x[10] = float("nan")
    x[11, ::2], x[11, 1::2] = 464.0, -0.0
    for shape in (x, x[4:5], x[7:10], x[9:11], x[5:7]):
        check(ops, shape, rows)
        check(ops, shape.to(torch.bfloat16), rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pitch,first", [(208, 0), (200, 0), (201, 1), (195, 3)])
def test_rows_of_any_pitch_and_place(ops, pitch, first, dtype, rows):
    wide = values(40, pitch, dtype, pitch).cuda()
    x = wide[:, first:first + 192]
    codes, scales = run(ops, x, rows)
    want, s = blocks(x.cpu(), rows)
    assert torch.equal(scales.double(), s) and same(codes, want)


def test_no_rows(ops):
    ops.quantize8(torch.empty(0, 64, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(1, 0, device="cuda"), torch.empty(0, 64, device="cuda"))


def test_refusals(ops):
    x = torch.ones(4, 64, device="cuda")
    codes, scales = torch.empty(4, 64, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(1, 4, device="cuda")
    ops.quantize8(codes, scales, x)
    wide = torch.empty(4, 128, dtype=torch.uint8, device="cuda")
    for c, s, v, rows in ((codes, scales, x, 2), (codes.view(torch.uint8), scales, x, 1), (codes, scales.double(), x, 1), (codes, scales, x.half(), 1),
                          (codes, scales[:, :3], x, 1), (codes, scales, x, 128), (codes, scales, x[:, :48], 1), (codes, scales, x.cpu(), 1),
                          (wide[:, :64].view(E4M3), scales, x, 1), (codes, scales, x.t().contiguous().t(), 1), (codes[:, :8], scales, x[:, :8], 1),
                          (torch.empty(264, dtype=torch.uint8, device="cuda")[8:].view(4, 64).view(E4M3), scales, x, 1)):
        with pytest.raises(ops.KernelError):
            ops.quantize8(c, s, v, rows)
