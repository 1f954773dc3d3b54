"""Probabilities at the smallest and the largest temperatures, with masked logits (-inf, NaN, the type's lowest value) in the rows. The rule and its bound are
those of the other settings."""
import numpy as np
import pytest
import torch

from test_draft_verify_gpu import check_probabilities, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def rows(vocab, lowest):
    torch.manual_seed(vocab)
    x = torch.randn(6, vocab) * 3
    x[1, ::3] = float("-inf")
    x[2, 1::2] = float("nan")
    x[3, vocab // 2:] = torch.finfo(torch.float32).min if lowest else -1e4
    x[4, 2:] = float("-inf")
    x[5] = x[5].round() + 0.0                                 # equal ones (without -0, which stands behind +0)
    return x


@pytest.mark.parametrize("vocab", [7, 600, 20000])
@pytest.mark.parametrize("top_k", [0, 3, 300])
@pytest.mark.parametrize("temperature", [1e-3, 1e-6, 5e-8, 4e-8, 3e-8, 1e-8, 7e-9, 1e-12, 1e-20, 1e-30, 1e-37, 1.2e-38, 4e-39, 1e-41, 1e-44])
def test_small_temperatures(ops, vocab, top_k, temperature):  # noqa: F811
    check_probabilities(ops, rows(vocab, True), float(np.float32(temperature)), top_k)


@pytest.mark.parametrize("vocab", [7, 600, 20000])
@pytest.mark.parametrize("top_k", [0, 3, 300])
@pytest.mark.parametrize("temperature", [50.0, 1e4, 1e10, 1e30, 1e36, 1e37, 3e38])
def test_large_temperatures(ops, vocab, top_k, temperature):  # noqa: F811
    check_probabilities(ops, rows(vocab, temperature < 1e34), float(np.float32(temperature)), top_k)


@pytest.mark.parametrize("temperature", [1e-8, 0.7, 1e37])
def test_a_prefix_by_mass(ops, temperature):  # noqa: F811
    """Masked logits never enter a prefix: two equal best ones and nothing else that counts."""
    x = torch.full((1, 900), float("-inf"))
    x[0, 5], x[0, 77] = 2.0, 2.0
    check_probabilities(ops, x, float(np.float32(temperature)), 0, 0.75)
    check_probabilities(ops, x, float(np.float32(temperature)), 0, 0.25)


@pytest.mark.parametrize("vocab,top_k", [(600, 300), (600, 40), (20000, 9000)])
def test_signed_zeros_stand_as_the_sampler_has_them(ops, vocab, top_k):  # noqa: F811
    """+0 before -0, equal ones by their ids: the kept tokens are those that a draw can give."""
    x = torch.full((1, vocab), -1.0)
    x[0, ::2] = -0.0
    x[0, 1::4] = 0.0
    p = torch.empty(1, vocab, device="cuda")
    ops.probabilities(p, x.cuda(), 1.0, top_k)
    order = sorted(range(vocab), key=lambda i: (-float(x[0, i]), bool(torch.signbit(x[0, i])), i))
    kept = torch.zeros(vocab, dtype=torch.bool)
    kept[order[:top_k]] = True
    assert torch.equal(p[0].cpu() > 0, kept)
    tokens = torch.empty(20000, dtype=torch.int32, device="cuda")
    ops.sample(x.cuda().expand(20000, vocab).contiguous(), tokens, 1.0, top_k, 1.0, torch.arange(20000, dtype=torch.int32, device="cuda"),
               torch.zeros(20000, dtype=torch.int32, device="cuda"))
    assert bool(kept[tokens.cpu().long()].all())
