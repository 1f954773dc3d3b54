"""Attention over pages of 8 bits: which rows a NaN code reaches."""
import pytest
import torch

from numbers8 import PAGE
from test_attention8_gpu import call, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


@pytest.mark.parametrize("dim", [48, 64, 128, 256])
@pytest.mark.parametrize("new,nq", [(1, 4), (2, 2), (6, 2), (5, 6), (6, 8)])
@pytest.mark.parametrize("window", [0, 50, 64])
def test_a_nan_value_reaches_all_rows_that_see_it(ops, dim, new, nq, window):
    """Wherever its key lies: in a page of its own, beside the new tokens, beside a window's first key. Each row's other results stay as they were."""
    nkv, length = 2, 300
    c = make([(new, length), (new, 90)], nq, nkv, dim, seed=dim + new)
    clean = call(ops, c, nq, nkv, dim, new, window).view(-1, nq, dim)
    group = nq // nkv
    for key in (0, 100, 191, 192, 235, 244, 245, 249, 250, 251, 255, 256, 275, 293, 294, 295, 298, 299):
        page = int(c["table"][c["seq_slots"][0], key // PAGE])
        bad = {**c, "v": c["v"].clone()}
        bad["v"].view(torch.uint8)[page, 1, key % PAGE, 5] = 0xFF
        got = call(ops, bad, nq, nkv, dim, new, window).view(-1, nq, dim)
        for i in range(new):
            at = length - new + i
            sees = key <= at and (not window or key > at - window)
            hit = torch.isnan(got[i])
            assert int(hit.sum()) == (group if sees else 0) and bool(hit[group:, 5].all()) == sees, (key, i)
            assert torch.equal(torch.where(hit, 0.0, got[i]), torch.where(hit, 0.0, clean[i])), (key, i)
        assert torch.equal(got[new:], clean[new:])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_key_reaches_all_rows_that_see_it(ops, dim):
    new, nq, nkv, length, window = 4, 4, 2, 300, 60
    c = make([(new, length)], nq, nkv, dim, seed=dim)
    clean = call(ops, c, nq, nkv, dim, new, window).view(-1, nq, dim)
    for key in (230, 237, 238, 240, 255, 256, 280, 297, 299):
        page = int(c["table"][c["seq_slots"][0], key // PAGE])
        bad = {**c, "k": c["k"].clone()}
        bad["k"].view(torch.uint8)[page, 1, key % PAGE, 5] = 0x7F
        got = call(ops, bad, nq, nkv, dim, new, window).view(-1, nq, dim)
        for i in range(new):
            at = length - new + i
            sees = at - window < key <= at
            assert bool(torch.isnan(got[i, 2:]).all()) if sees else torch.equal(got[i], clean[i]), (key, i)
            assert torch.equal(got[i, :2], clean[i, :2])
