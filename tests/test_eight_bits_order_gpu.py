"""8-bit operators called directly after the one that makes what they read: nothing is read before it is written, called or captured."""
import pytest
import torch

from numbers8 import E4M3

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
