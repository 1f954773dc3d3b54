"""The tests' own e4m3 rounding against torch's conversion, and scales at their borders (CPU)."""
import pytest
import torch

from numbers8 import E4M3, F64, blocks, nearest, power, same


def test_rounding_is_that_of_the_type():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(5000, generator=g) * 10.0 ** e for e in (-4, -2, 0, 2)]).clamp(-448, 448)
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    codes = codes[torch.isfinite(codes)]
    ties = (codes.sort().values[1:] + codes.sort().values[:-1]) / 2
    for v in (x, codes, ties):
        assert same(nearest(v), v.to(E4M3).float())


@pytest.mark.parametrize("e", [-100, -30, 0, 60, 120])
def test_scales_at_their_borders(e):
    s = 2.0 ** e
    assert float(power(448.0 * s)) == s
    assert float(power(448.0 * s * (1 + 2.0 ** -23))) == 2 * s
    assert float(power(224.0 * s)) == max(s / 2, 2.0 ** -100)
    assert float(power(0.0)) == 2.0 ** -100


def test_blocks_of_what_is_not_finite():
    x = torch.ones(2, 32)
    x[0, 3], x[1, 5], x[1, 6] = float("inf"), float("nan"), -float("inf")
    v, s = blocks(x, 1)
    assert torch.isnan(v).nonzero().tolist() == [[0, 3], [1, 5], [1, 6]]
    assert s.shape == (1, 2) and bool((v[torch.isfinite(v)] * float(s[0, 0]) == 1).all()) and v.dtype == F64
