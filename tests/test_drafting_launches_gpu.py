"""The count of launched kernels against the kernel nodes of a captured call."""
import ctypes

import pytest
import torch

from test_work_spaces_gpu import attention_case, linear_case, verify_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def kernels(call):
    """(kernel nodes, what the library counted) of one captured call."""
    from tileinfer_b200.kernels import library
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = library.launch_count
    with torch.cuda.graph(graph):
        call()
    counted = library.launch_count - before
    driver, n = ctypes.CDLL("libcuda.so.1"), ctypes.c_size_t()
    handle = ctypes.c_void_p(graph.raw_cuda_graph())
    assert driver.cuGraphGetNodes(handle, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert driver.cuGraphGetNodes(handle, nodes, ctypes.byref(n)) == 0
    found = 0
    for node in nodes:
        kind = ctypes.c_int(-1)
        assert driver.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        found += kind.value == 0                              # CU_GRAPH_NODE_TYPE_KERNEL
    return found, counted


@pytest.mark.parametrize("n,out,k", [(1, 1024, 1024), (20, 1024, 4096), (8, 2048, 9216), (20, 37888, 256), (64, 4096, 256), (9, 256 * 148, 1024), (300, 1024, 512)])
def test_products(ops, n, out, k):
    found, counted = kernels(linear_case(ops, n, out, k, 1)[0])
    assert found == counted


def test_a_product_of_unaligned_rows(ops):
    """Rows that do not go through shared memory have no join."""
    codes = torch.zeros(1024, 512, dtype=torch.int32, device="cuda")
    scales = torch.ones(32, 1024, dtype=torch.bfloat16, device="cuda")
    x, y = torch.zeros(20, 4097, dtype=torch.bfloat16, device="cuda")[:, 1:], torch.empty(20, 1024, dtype=torch.bfloat16, device="cuda")
    found, counted = kernels(lambda: ops.linear4(y, x, codes, scales))
    assert found == counted == 1


@pytest.mark.parametrize("seqs", [1, 512, 513, 1100])
def test_attention(ops, seqs):
    found, counted = kernels(attention_case(ops, seqs, 2, 70, 1)[0])
    assert found == counted


def test_a_test_of_drafts_with_a_work_space(ops):
    call, _ = verify_case(ops, 5, 1)
    inner, ws = ops.verify_drafts, torch.zeros(ops.verify_drafts_workspace(5), dtype=torch.uint8, device="cuda")
    ops.verify_drafts = lambda *a: inner(*a, workspace=ws)
    try:
        found, counted = kernels(call)
    finally:
        ops.verify_drafts = inner
    assert found == counted == 1
