"""What infinities and NaN among a token's own visible scores and values come to: what the definition makes of them, in the rows that see them alone."""
import pytest
import torch

from test_attention_few_gpu import call, make, reference

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def spoiled(where, what, key, nq=4, nkv=2, dim=64, runs=((3, 700), (2, 90), (1, 5000))):
    """A case whose key (or value, or query) at position ``key`` of every sequence's first KV head is ``what``."""
    c = make(runs, nq, nkv, dim, 3)
    for b, (_, length) in enumerate(runs):
        at = min(key, length - 1)
        page = int(c["table"][int(c["seq_slots"][b]), at // 64])
        if where == "q":
            c["q"][int(c["cu"][b]), 0] = what
        else:
            c[where][page, 0, at % 64] = what
    return c


def check(ops, c, nq, nkv, dim, window=0):
    got = call(ops, c, nq, nkv, dim, 3, window).to(F64)
    want, bound = reference(c, dim ** -0.5, window)
    finite = torch.isfinite(want)
    assert not bool(finite.all())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert bool(((got - want).abs() <= bound)[finite].all())


@pytest.mark.parametrize("dim,nq,nkv", [(64, 4, 2), (32, 4, 2), (256, 4, 2), (128, 32, 2)])
@pytest.mark.parametrize("where,what", [("k", float("nan")), ("v", float("nan")), ("v", float("inf")), ("q", float("nan")), ("k", float("inf"))])
@pytest.mark.parametrize("key", [0, 63])
def test_they_reach_the_rows_that_see_them(ops, dim, nq, nkv, where, what, key):
    check(ops, spoiled(where, what, key, nq, nkv, dim), nq, nkv, dim)


@pytest.mark.parametrize("dim,nq,nkv", [(64, 4, 2), (256, 4, 2), (128, 32, 2)])
@pytest.mark.parametrize("where,what", [("k", float("nan")), ("q", float("nan")), ("k", float("-inf"))])
def test_in_a_runs_last_key_or_query(ops, dim, nq, nkv, where, what):
    """Every sequence's last position, which its last token alone sees."""
    check(ops, spoiled(where, what, 10 ** 6, nq, nkv, dim), nq, nkv, dim)


@pytest.mark.parametrize("dim,nq,nkv", [(16, 4, 2), (64, 4, 2), (80, 8, 1), (96, 12, 2), (256, 4, 2), (128, 32, 2), (128, 64, 2), (32, 60, 2)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window", [0, 1, 2, 70])
def test_a_value_that_some_tokens_of_a_run_do_not_see(ops, dim, nq, nkv, what, window):
    """A drafted token's own value, which the tokens before it do not see; with a window the first values, which the later tokens do not see any more."""
    runs = ((3, 700), (2, 90), (1, 5000), (3, 65), (3, 3))
    check(ops, spoiled("v", what, 10 ** 6, nq, nkv, dim, runs), nq, nkv, dim, window)
    c = spoiled("v", what, 10 ** 6, nq, nkv, dim, runs)
    for b, (new, length) in enumerate(runs):
        for at in (length - 2, length - window - 1):          # the middle of a run; the last that its last token but one sees, not its last
            if at >= 0:
                c["v"][int(c["table"][int(c["seq_slots"][b]), at // 64]), 1 % nkv, at % 64, 3] = what
    check(ops, c, nq, nkv, dim, window)
