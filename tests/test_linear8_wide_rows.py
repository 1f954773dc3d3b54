"""Products of few tokens whose rows are so long that a block of eight warps has no room for the tokens' codes: the kernel for more tokens takes them."""
import pytest
import torch

from tileinfer_b200.kernels import library

COLUMNS = (44048, 45056, 50000, 65536, 77824)


@pytest.mark.parametrize("k", COLUMNS)
@pytest.mark.parametrize("out", [16, 512, 4096, 131072])
def test_the_kernel_that_takes_them(k, out):
    """One to four tokens of up to 44,032 columns are quantised in the product's own blocks, those of longer rows ahead (sixteen bytes at a time)."""
    need = library.lib().ti_linear8_workspace
    for n in (1, 4):
        assert need(n, out, 44032, 0) == 0
        assert need(n, out, k, 0) == n * k + -(-4 * n * -(-k // 128) // 16) * 16


@pytest.mark.gpu
@pytest.mark.parametrize("k", COLUMNS + (44032, 90000))
@pytest.mark.parametrize("n", [1, 4, 8])
@pytest.mark.parametrize("out", [37, 1000])
def test_long_rows(n, out, k):
    from tileinfer_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(k + n)
    w, x = torch.randn(out, k, device="cuda", generator=g).bfloat16(), torch.randn(n, k, device="cuda", generator=g).bfloat16()
    codes, scales = torch.empty(out, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.empty(-(-k // 128), -(-out // 128), device="cuda")
    made, x_scales = torch.empty(n, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.empty(-(-k // 128), n, device="cuda")
    ops.quantize8(codes, scales, w, 128)
    ops.quantize8(made, x_scales, x)
    wide = lambda c, s, rows: c.float().double() * s.t().double().repeat_interleave(rows, 0)[:c.shape[0]].repeat_interleave(128, 1)[:, :k]  # noqa: E731
    xs, ws = wide(made, x_scales, 1), wide(codes, scales, 128)
    want, size = xs @ ws.t(), xs.abs() @ ws.abs().t()
    # products of codes are exact in 32 bits; a sum of k of them is off by at most k 2^-23 of their sizes, each group's scale and the join by a few 2^-23 more, and y is rounded once
    bound = size * (k + 16) * 2.0 ** -23 + want.abs() * 2.0 ** -8
    for args in ((x, codes, scales), (made, codes, scales, x_scales)):
        y = torch.full((n + 1, out), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.linear8(y[:n], *args)
        assert bool(((y[:n].double() - want).abs() <= bound).all()) and bool((y[n] == 7).all())
    # the sums themselves, tighter: a group's sum is off by at most 16 steps of 2^-23 of its size, the at most 704 groups are added with 2^-24 of the whole each:
    # 704 2^-24 + 2^-19 < 2^-14 (a lost group is some 2^-9)
    y = torch.empty(n, out, device="cuda")
    ops.linear8(y, x, codes, scales, None, ops.EPI_F32_OUT)
    assert bool(((y.double() - want).abs() <= 2.0 ** -14 * size).all())
    ops.check_status()
