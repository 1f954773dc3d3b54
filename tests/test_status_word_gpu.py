"""The word that kernels with bounded waits report to, where the first call that needs it is one that is being captured."""
import subprocess
import sys

import pytest
import torch

from test_work_spaces_gpu import CASES, capture, results, same

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops():
    from tileinfer_b200.kernels import ops
    ops.status_word()
    held, ops._status = ops._status, None                     # as in a program that has made no call yet
    yield ops
    ops._status = held


@pytest.mark.parametrize("kind", ["linear4", "attention"])
def test_first_made_while_capturing(ops, kind):
    case = CASES[kind](ops, 1)
    held = []
    before = capture(lambda: held.extend(torch.full((1 << 17,), -1, dtype=torch.int32, device="cuda") for _ in range(8)))
    before.replay()
    torch.cuda.synchronize()
    held.clear()                                              # the graph's memory holds something else
    graph = capture(case[0], pool=before.pool())
    ops.check_status()                                        # nothing has run yet: nothing to report
    graph.replay()
    got = [o.clone() for o in case[1]]
    ops.check_status()
    assert same(got, results(case))
    # A report stands until it is read, whatever graphs are replayed meanwhile.
    ops.status_word().fill_(1 << 28)
    graph.replay()
    with pytest.raises(ops.KernelError, match="gave up"):
        ops.check_status()
    ops.check_status()


def test_the_first_call_of_a_program_is_captured():
    """In a process of its own: nothing of the library has run before the capture."""
    program = """
import sys
sys.path[:0] = ["tests", "."]
import torch
from tileinfer_b200.kernels import ops
from test_work_spaces_gpu import attention_case, capture
call, outs = attention_case(ops, 2, 5, 9000, 1)
graph = capture(call)
graph.replay()
got = outs[0].clone()
ops.check_status()
call()
assert torch.equal(got, outs[0]) and bool(got.any())
print("same")
"""
    import conftest
    done = subprocess.run([sys.executable, "-c", program], cwd=conftest.ROOT, capture_output=True, text=True, timeout=300)
    assert done.stdout.strip() == "same", done.stderr[-2000:]
