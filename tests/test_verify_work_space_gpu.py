"""The work space that a caller brings to the test of drafts."""
import pytest
import torch

from test_work_spaces_gpu import results, same, verify_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def with_space(ops, ws, seqs, seed, k=4, vocab=5000):
    """The call of ``verify_case`` with ``ws``."""
    call, outs = verify_case(ops, seqs, seed, k, vocab)
    inner = ops.verify_drafts
    ops.verify_drafts = lambda *a: inner(*a, workspace=ws)
    try:
        call()
    finally:
        ops.verify_drafts = inner
    return outs


def test_a_work_space_of_ones_own(ops):
    """Calls of as many sequences and of fewer, in any order, from one zeroed work space; also from the one that the library keeps."""
    ws = torch.zeros(ops.verify_drafts_workspace(70) + 24, dtype=torch.uint8, device="cuda")
    for seed, seqs in enumerate((70, 3, 70, 1, 33, 69, 70)):
        want = results(verify_case(ops, seqs, seed))
        assert same(with_space(ops, ws, seqs, seed), want)


def test_graphs_with_work_spaces_of_their_own(ops):
    a, b = (torch.zeros(ops.verify_drafts_workspace(8), dtype=torch.uint8, device="cuda") for _ in range(2))
    case = verify_case(ops, 8, 1)
    want = results(case)
    inner, graphs = ops.verify_drafts, []
    for ws in (a, b):
        ops.verify_drafts = lambda *args, ws=ws: inner(*args, workspace=ws)
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                case[0]()
            graphs.append(graph)
        finally:
            ops.verify_drafts = inner
    for graph in reversed(graphs):
        for _ in range(2):
            for o in case[1]:
                o.fill_(-3)
            graph.replay()
            assert same(case[1], want)


def test_refused_work_spaces(ops):
    need = ops.verify_drafts_workspace(5)
    good = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    for ws in (good[:need - 1], good[1:], good.cpu(), good[:need // 4 * 4].view(torch.int32), torch.zeros(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ops.KernelError, match="work space"):
            with_space(ops, ws, 5, 0)
