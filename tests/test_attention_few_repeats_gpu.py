"""The same bits from the same call, many times over, at sizes where tiles come from memory and every place of the ring is used again and again.

A copy that overtakes a read of the tile before it in the same place changes a few rows of an item now and then, so the calls are many and large."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def batch(seqs, new, length, nq, nkv, dim, seed=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-length // 64)
    k, v = (torch.randn(seqs * pages, nkv, 64, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(seqs * new, nq, dim, generator=g, device="cuda").to(torch.bfloat16)
    int32 = lambda t: torch.as_tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.randperm(seqs * pages, generator=g, device="cuda").to(torch.int32).view(seqs, pages)
    return q, k, v, table, int32(range(seqs)), int32(range(0, seqs * new + 1, new)), int32([length] * seqs)


@pytest.mark.parametrize("seqs,new,length,nq,nkv,dim", [(64, 4, 1024, 32, 8, 128), (1, 5, 65531, 32, 8, 128), (8, 8, 8192, 64, 8, 128), (64, 2, 2048, 16, 8, 64),
                                                        (48, 2, 1000, 8, 4, 256), (64, 4, 2048, 16, 8, 96), (64, 4, 4096, 8, 8, 32)])
def test_the_same_bits(seqs, new, length, nq, nkv, dim):
    from tileinfer_b200.kernels import ops
    args = batch(seqs, new, length, nq, nkv, dim)
    outs = [torch.empty(seqs * new, nq * dim, dtype=torch.bfloat16, device="cuda") for _ in range(16)]
    for _ in range(12):
        for out in outs:
            ops.attention_few(out, *args, dim ** -0.5, nq, nkv, dim, 64, new)
        assert all(torch.equal(out, outs[0]) for out in outs[1:])
    ops.check_status()
    # And the right ones: every item of a few sequences, from the definition.
    q, k, v, table = args[:4]
    for b in {0, seqs // 2, seqs - 1}:
        keys, values = (t[table[b].long()].permute(1, 0, 2, 3).reshape(nkv, -1, dim)[:, :length].double() for t in (k, v))
        z = q[b * new:(b + 1) * new].double().view(new, nkv, nq // nkv, dim).permute(1, 2, 0, 3) @ keys[:, None].transpose(-1, -2) * dim ** -0.5
        hidden = torch.arange(length, device="cuda")[None, :] > length - new + torch.arange(new, device="cuda")[:, None]
        p = torch.softmax(z.masked_fill(hidden, float("-inf")), -1)
        want, size = p @ values[:, None], p @ values[:, None].abs()
        got = outs[0][b * new:(b + 1) * new].double().view(new, nkv, nq // nkv, dim).permute(1, 2, 0, 3)
        rough = float(z.abs().max()) * dim * 2.0 ** -23      # a score's sum, twice in a weight and its denominator
        assert bool(((got - want).abs() <= size * (2.0 ** -8 + 2.5 * rough + 2.0 ** -18) + want.abs() * 2.0 ** -8).all())
