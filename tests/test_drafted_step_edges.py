"""Calls at the edges of what include/strasgpt_kernels.h allows of a step over
drafted tokens: threads, captured and replayed steps, values at the ends of
their ranges, buffers that are shared.
"""
import os
import subprocess
import sys

import numpy as np
import pytest
from test_drafted_step import BF16, F32, check_sample, dtype

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


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("vocab", [70, 3001, 40000])
@pytest.mark.parametrize("rows", [7, 300])
def test_sample_distances_beyond_fp32(cuda, type_, vocab, rows):
    """Logits whose distance from the largest overflows fp32, at temperatures
    that give them a weight all the same: the largest and the lowest value of
    the type; masks of the lowest value under ordinary logits. With few rows
    (clusters) and with many (under top-k, a block each)."""
    torch = cuda
    inf = float("inf")
    x = torch.full((7, vocab), -inf, device="cuda", dtype=dtype(torch, type_))
    low, high = torch.finfo(x.dtype).min, torch.finfo(x.dtype).max
    x[0, 5], x[0, 50:60], x[0, 69] = high, 1.0, low
    x[1, 0:3] = torch.tensor([low, 1.0, high])
    x[2] = low
    x[2, 11:40] = torch.arange(29, device="cuda") / 4
    x[3] = 2e38
    x[3, ::2] = -2e38
    x[4, ::3] = high
    x[4, 1::3] = low
    x[5] = torch.linspace(low / 2, high / 2, vocab, device="cuda")   # the difference just fits
    x[6] = torch.linspace(float(low) * 0.9, float(high) * 0.9, vocab, device="cuda",
                          dtype=torch.float64).to(x.dtype)
    x = x.repeat((rows + 6) // 7, 1)[:rows]
    rng = np.random.RandomState(vocab)
    for heat in (inf, 1e38, 3e38, 2e37, 1e36, 1.0):
        for f in (dict(), dict(top_k=2), dict(top_k=40, top_p=0.97), dict(top_p=0.7),
                  dict(min_p=0.01), dict(top_k=300, min_p=0.3)):
            check_sample(torch, x, heat=heat, u=rng.uniform(0.01, 0.99, rows).astype(np.float32),
                         **f)
