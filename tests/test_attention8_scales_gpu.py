"""Attention over pages of 8 bits whose value scales lie far apart: a page of zeros has 2^-100, others up to 2^120. Bounds as in test_attention8_gpu.py."""
import pytest
import torch

from numbers8 import F64
from test_attention8_gpu import call, make, reference

pytestmark = pytest.mark.gpu
HEADS = [(8, 2, 128), (2, 2, 64), (4, 1, 256)]


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def right(ops, c, nq, nkv, dim, new, window=0):
    got = call(ops, c, nq, nkv, dim, new, window)
    want, bound = reference(c, dim ** -0.5, window, 11)
    off = (got.to(F64) - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


def pages(c, b):
    return c["table"][int(c["seq_slots"][b]), :-(-int(c["lens"][b]) // 64)].long()


@pytest.mark.parametrize("nq,nkv,dim", HEADS)
@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("large", [0, 25, 33, 34, 40, 80, 110])
@pytest.mark.parametrize("order", ["zeros first", "zeros last", "in turn"])
def test_pages_of_zeros_beside_others(ops, nq, nkv, dim, new, large, order):
    """Their keys have as much weight as others'; their values are zero."""
    runs = [(new, 1300), (new, 129), (new, 9000)]
    c = make(runs, nq, nkv, dim, seed=large)
    for b, (_, length) in enumerate(runs):
        p = pages(c, b)
        zeros = p[:len(p) // 2] if order == "zeros first" else p[len(p) // 2:] if order == "zeros last" else p[::2]
        c["vs"][p] = 2.0 ** large
        c["vs"][zeros] = 2.0 ** -100
        length_in = torch.arange(len(p) * 64).view(-1, 64) < length
        for i, page in enumerate(p.tolist()):
            if page in zeros.tolist():
                c["v"].view(torch.uint8)[page][:, length_in[i]] = 0
    right(ops, c, nq, nkv, dim, new)


@pytest.mark.parametrize("nq,nkv,dim", HEADS)
@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("low,high", [(-100, 110), (-100, -60), (60, 110), (-20, 100)])
def test_scales_anywhere_in_the_range(ops, nq, nkv, dim, new, low, high):
    c = make([(new, 700), (new, 20000), (new, 64)], nq, nkv, dim, seed=high)
    c["vs"] = torch.exp2(torch.randint(low, high + 1, c["vs"].shape, generator=torch.Generator().manual_seed(new)).float())
    right(ops, c, nq, nkv, dim, new)
    right(ops, c, nq, nkv, dim, new, 300)


@pytest.mark.parametrize("large", [-100, 0, 34, 110])
def test_a_long_run_of_zeros_and_one_ordinary_page(ops, large):
    """The ordinary page is the last; and scores that grow along the run, so that the weights' base follows them."""
    nq, nkv, dim = 4, 2, 128
    c = make([(1, 30000), (3, 14000)], nq, nkv, dim, seed=1)
    for b in range(2):
        p = pages(c, b)
        c["vs"][p] = 2.0 ** -100
        c["v"].view(torch.uint8)[p[:-1]] = 0
        c["vs"][p[-1]] = 2.0 ** large
        c["ks"][p] *= torch.linspace(0.01, 4, len(p))[:, None]
    right(ops, c, nq, nkv, dim, 3)


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** 115])
def test_all_scales_at_an_end_of_the_range(ops, size):
    c = make([(1, 3000), (4, 40), (2, 300)], 8, 4, 64, seed=2)
    c["vs"].fill_(size)
    right(ops, c, 8, 4, 64, 4)


@pytest.mark.parametrize("by", [30.0, 60.0, 100.0])
def test_pages_of_zeros_that_take_the_weight(ops, by):
    """Scores of a page of zeros are ``by`` powers of two above the others': what is left of the others' values is that much smaller."""
    nq, nkv, dim = 2, 2, 64
    c = make([(1, 640)], nq, nkv, dim, seed=3)
    p = pages(c, 0)
    c["q"].fill_(1.0)
    c["k"] = torch.zeros_like(c["k"].float()).to(c["k"].dtype)
    c["ks"].fill_(1.0)
    c["k"][p[4]] = torch.tensor(4.0).to(c["k"].dtype)
    c["ks"][p[4]] = by * 0.6931 / (4.0 * dim * dim ** -0.5)
    c["vs"][p] = 2.0 ** 40
    c["vs"][p[4]] = 2.0 ** -100
    c["v"].view(torch.uint8)[p[4]] = 0
    right(ops, c, nq, nkv, dim, 1)
