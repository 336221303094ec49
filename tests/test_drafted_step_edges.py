"""Calls at the edges of what include/strasgpt_kernels.h allows of a step over
drafted tokens: threads, captured and replayed steps, values at the ends of
their ranges, buffers that are shared.
"""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_first_calls_from_two_threads(cuda):
    """In a process of its own: the first calls of two host threads, with
    vocabularies whose rows need 100 and 200 KB of shared memory, are served,
    and so are all later ones."""
    program = """
import threading, torch
from strasgpt_b200 import runtime
L = runtime.lib()
u = torch.full((1,), 0.5, device="cuda")
xs = [torch.randn(1, v, device="cuda") for v in (160000, 320000)]
out = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in xs]
torch.cuda.synchronize()
ready, status = threading.Barrier(2), []
def calls(i):
    ready.wait()
    for _ in range(200):
        status.append(L.strasgpt_k_sample(
            xs[i].data_ptr(), 0, xs[i].shape[1], 1, xs[i].shape[1], None, None, None, None,
            u.data_ptr(), out[i].data_ptr(), None, None, None))
threads = [threading.Thread(target=calls, args=(i,)) for i in (0, 1)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert status == [0] * 400, status
"""
    for _ in range(2):
        subprocess.run([sys.executable, "-c", program], cwd=ROOT, check=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=ROOT))
