"""8-bit operators called directly after the one that makes what they read: nothing is read before it is written, called or captured."""
import pytest
import torch

from numbers8 import E4M3, PAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


@pytest.mark.parametrize("n,given", [(1, False), (8, False), (5, True), (20, True), (300, True)])
@pytest.mark.parametrize("out,k", [(256, 512), (4096, 8192)])
def test_products_directly_after_their_weights(ops, n, given, out, k):
    """One place for the codes takes two matrices' in turn; the product right behind sees its own."""
    g = torch.Generator().manual_seed(n)
    ws = [torch.randn(out, k, generator=g).bfloat16().cuda() * size for size in (1.0, 64.0)]
    x = torch.randn(n, k, generator=g).bfloat16().cuda()
    codes, scales = torch.empty(out, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(-(-k // 128), -(-out // 128), device="cuda")
    x_scales = None
    if given:
        made, x_scales = torch.empty(n, k, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(-(-k // 128), n, device="cuda")
        ops.quantize8(made, x_scales, x)
        x = made
    want = []
    for w in ws:
        ops.quantize8(codes, scales, w, 128)
        torch.cuda.synchronize()
        want.append(torch.empty(n, out, dtype=torch.bfloat16, device="cuda"))
        ops.linear8(want[-1], x, codes, scales, x_scales)
        torch.cuda.synchronize()

    def turns(outs):
        for i, y in enumerate(outs):
            ops.quantize8(codes, scales, ws[i % 2], 128)
            ops.linear8(y, x, codes, scales, x_scales)

    outs = [torch.zeros(n, out, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        turns(outs)
        stream.synchronize()
        assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(outs))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            turns(outs)
        for _ in range(10):
            for y in outs:
                y.zero_()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(outs))


@pytest.mark.parametrize("written", [1, 2, 64, 200, 1000])
@pytest.mark.parametrize("attending", [1, 3])
def test_attention_of_fewer_tokens_than_were_just_written(ops, written, attending):
    """A run's keys and values go into the cache and its last tokens alone attend, right behind; two runs take one place in turn."""
    nq, nkv, dim, seqs = 8, 4, 128, 6
    attending = min(attending, written)
    pages = -(-(written + 70) // PAGE)
    g = torch.Generator().manual_seed(written)
    table = torch.randperm(seqs * pages, generator=g).to(torch.int32).view(seqs, pages).cuda()
    slots = torch.arange(seqs, dtype=torch.int32).cuda()
    ranges = [(torch.arange(seqs + 1) * t).to(torch.int32).cuda() for t in (written, attending)]
    lens = torch.full((seqs,), written + 70, dtype=torch.int32).cuda()
    new = [[torch.randn(seqs * written, nkv, dim, generator=g).bfloat16().cuda() * size for _ in "kv"] for size in (1.0, 3.0)]
    q = torch.randn(seqs * attending, nq, dim, generator=g).bfloat16().cuda()
    k, v = (torch.zeros(seqs * pages, nkv, PAGE, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in "kv")
    ks, vs = (torch.ones(seqs * pages, nkv, device="cuda") for _ in "kv")

    def write(i):
        ops.cache_write8(k, v, ks, vs, *new[i % 2], table, slots, ranges[0], lens, written)

    def attend(out):
        ops.attention8(out, q, k, v, ks, vs, table, slots, ranges[1], lens, dim ** -0.5, nq, nkv, dim, PAGE, attending)

    outs = [torch.zeros(seqs * attending, nq * dim, dtype=torch.bfloat16, device="cuda") for _ in range(8)]

    def fresh():
        for t in (k, v):
            t.view(torch.uint8).zero_()
        ks.fill_(1.0), vs.fill_(1.0)

    def turns(wait=False):
        for i, out in enumerate(outs):
            write(i)
            if wait:
                torch.cuda.synchronize()
            attend(out)
            if wait:
                torch.cuda.synchronize()

    fresh()
    turns(wait=True)
    want = [out.clone() for out in outs]
    assert not torch.equal(want[0], want[1])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        fresh()
        turns()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            fresh()
            turns()
        for _ in range(5):
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    ops.check_status()
