"""Calls of two Python threads on one stream: whatever order their kernels come in, each gets the bits of its own call."""
import threading

import pytest
import torch

from test_work_spaces_gpu import CASES, results

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", CASES)
def test_two_threads_on_one_stream(kind):
    from tileinfer_b200.kernels import ops
    cases = [CASES[kind](ops, seed) for seed in (1, 2, 3)]
    want = [results(c) for c in cases]
    wrong, start = [], threading.Barrier(len(cases))

    def work(i):
        call, outs = cases[i]
        start.wait()
        for _ in range(20):
            seen = []
            for _ in range(10):
                call()
                seen.append([o.clone() for o in outs])
            wrong.extend(i for got in seen if not all(torch.equal(a, b) for a, b in zip(got, want[i])))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
