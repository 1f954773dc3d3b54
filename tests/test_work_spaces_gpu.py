"""The work space that a call brings along by itself: calls captured in CUDA graphs hold none that another call, graph or stream uses, and none that is
given back before the graph is.

Results are compared bit for bit with the same calls made one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def verify_case(ops, seqs, seed, k=4, vocab=5000):
    """(call, outputs): a test of drafts with outputs of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.softmax(2 * torch.randn(seqs, k + 1, vocab, generator=g, device="cuda"), -1)
    q = torch.softmax(p[:, :k].log() + 0.7 * torch.randn(seqs, k, vocab, generator=g, device="cuda"), -1)
    drafts = torch.multinomial(q.reshape(-1, vocab), 1, generator=g).view(seqs, k).to(torch.int32)
    u = torch.randint(0, 1 << 24, (seqs, k + 1), generator=g, device="cuda").float() * 2.0 ** -24
    outs = torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(seqs, k + 1, dtype=torch.int32, device="cuda")
    return (lambda: ops.verify_drafts(*outs, p, q, drafts, u)), outs


def linear_case(ops, n, out, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-1 << 31, (1 << 31) - 1, (out, k // 8), generator=g, device="cuda").to(torch.int32)
    scales = (torch.rand(k // 128, out, generator=g, device="cuda") * 0.01).to(torch.bfloat16)
    x = torch.randn(n, k, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.zeros(n, out, dtype=torch.bfloat16, device="cuda")
    return (lambda: ops.linear4(y, x, codes, scales)), (y,)


def attention_case(ops, seqs, new, length, seed, nq=8, nkv=2, dim=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-length // 64)
    k, v = (torch.randn(seqs * pages, nkv, 64, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(seqs * new, nq, dim, generator=g, device="cuda").to(torch.bfloat16)
    int32 = lambda t: torch.as_tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    table, slots = int32(range(seqs * pages)).view(seqs, pages), int32(range(seqs))
    cu, lens = int32(range(0, seqs * new + 1, new)), int32([length] * seqs)
    out = torch.zeros(seqs * new, nq * dim, dtype=torch.bfloat16, device="cuda")
    return (lambda: ops.attention_few(out, q, k, v, table, slots, cu, lens, dim ** -0.5, nq, nkv, dim, 64, new)), (out,)


CASES = {"verify": lambda ops, seed: verify_case(ops, 6, seed), "linear4": lambda ops, seed: linear_case(ops, 20, 1024, 4096, seed),
         "attention": lambda ops, seed: attention_case(ops, 2, 5, 9000, seed)}
LARGER = {"verify": lambda ops: verify_case(ops, 300, 9), "linear4": lambda ops: linear_case(ops, 40, 4096, 4096, 9),
          "attention": lambda ops: attention_case(ops, 3, 33, 5000, 9)}


def results(case):
    call, outs = case
    call()
    got = [o.clone() for o in outs]
    for o in outs:
        o.fill_(-3)
    return got


def capture(call, stream=None, pool=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, pool=pool):
        call()
    return graph


def same(outs, want):
    return all(torch.equal(a, b) for a, b in zip(outs, want))


def scribble():
    """Freed memory comes back with something else in it."""
    junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(24)]
    torch.cuda.synchronize()
    return junk


@pytest.mark.parametrize("kind", CASES)
def test_the_second_graph_of_two_alone(ops, kind):
    """Two graphs with calls of the same size; the second is replayed first, and again after the first one is gone."""
    a, b = CASES[kind](ops, 1), CASES[kind](ops, 2)
    want = results(b)
    # Memory that a graph before them has filled with something else.
    held = []
    before = capture(lambda: held.extend(torch.full((1 << 17,), -1, dtype=torch.int32, device="cuda") for _ in range(8)))
    before.replay()
    torch.cuda.synchronize()
    held.clear()
    first, second = capture(a[0], pool=before.pool()), capture(b[0], pool=before.pool())
    for _ in range(2):
        for o in b[1]:
            o.fill_(-3)
        second.replay()
        assert same(b[1], want)
    del first
    torch.cuda.empty_cache()
    junk = scribble()
    for o in b[1]:
        o.fill_(-3)
    second.replay()
    assert same(b[1], want) and len(junk) == 24


@pytest.mark.parametrize("kind", CASES)
def test_graphs_side_by_side(ops, kind):
    """Two graphs replayed on two streams at once."""
    a, b = CASES[kind](ops, 3), CASES[kind](ops, 4)
    want_a, want_b = results(a), results(b)
    graphs, streams = (capture(a[0]), capture(b[0])), (torch.cuda.Stream(), torch.cuda.Stream())
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert same(a[1], want_a) and same(b[1], want_b)


@pytest.mark.parametrize("kind", CASES)
def test_a_stream_that_captured_goes_on_to_larger_calls(ops, kind):
    """A call on a stream, a capture there, then a larger call there, which needs more."""
    a, larger = CASES[kind](ops, 5), LARGER[kind](ops)
    want = results(a)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a[0]()
    graph = capture(a[0], stream)
    with torch.cuda.stream(stream):
        larger[0]()
    torch.cuda.synchronize()
    junk = scribble()
    for o in a[1]:
        o.fill_(-3)
    graph.replay()
    torch.cuda.synchronize()
    assert same(a[1], want) and all(bool((j == -1).all()) for j in junk)


@pytest.mark.parametrize("kind", CASES)
def test_between_a_graphs_replays(ops, kind):
    """Calls outside the graph, between its replays, on the stream that it was captured on."""
    a, b = CASES[kind](ops, 6), CASES[kind](ops, 7)
    want_a, want_b = results(a), results(b)
    graph = capture(a[0])
    for _ in range(3):
        for o in (*a[1], *b[1]):
            o.fill_(-3)
        b[0]()
        graph.replay()
        assert same(a[1], want_a) and same(b[1], want_b)
