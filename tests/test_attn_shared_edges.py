"""strasgpt_k_attn_shared (include/strasgpt_kernels.h) where device memory holds numbers
that no caller means: whatever `first` says, nothing outside the call's rows is read or
written. Tolerances are test_attn_shared's.
"""
import numpy as np
import pytest
import test_attn_shared as shared
from test_drafted_step_host import run_program

F32, BF16 = shared.F32, shared.BF16
LOWEST, HIGHEST = -(1 << 31), (1 << 31) - 1


def test_any_first_gives_rows_of_the_call(tmp_path):
    """Every pair of neighbouring entries of `first`, the ends of 32 bits among them,
    against the same cut in wider numbers."""
    run_program(tmp_path, r"""
#include "attn_tree.h"
#include <algorithm>
#include <climits>
#include <cstdio>
int main() {
  const int values[] = {INT_MIN, INT_MIN + 1, INT_MIN + 5, INT_MIN + 9, -(1 << 30), -9, -1, 0, 1, 5,
                        7, 8, 9, 1 << 30, INT_MAX - 1, INT_MAX};
  for (int tokens : {1, 8, INT_MAX})
    for (int most : {1, 6, 1024})
      for (int from : values)
        for (int to : values) {
          int token0 = -1, t = -1;
          sg::cut_tokens(from, to, tokens, most, &token0, &t);
          const long long a = std::min(std::max((long long)from, 0ll), (long long)tokens);
          const long long n = std::min((long long)to, (long long)tokens) - a;
          const long long want = std::min(std::max(n, 0ll), (long long)most);
          if (token0 != a || t != want || t < 0 || (long long)token0 + t > tokens) {
            printf("first %d, %d of %d tokens, %d at most: rows %d to %d, not %lld to %lld\n", from,
                   to, tokens, most, token0, token0 + t, a, a + want);
            return 1;
          }
        }
  return 0;
}
""")


def between_margins(torch, size, value=0x5A):
    """`size` bytes on 256 within a larger buffer, and that buffer, all of one pattern."""
    margin = 16384
    whole = torch.full((margin + (size + 255) // 256 * 256 + margin,), value, device="cuda",
                       dtype=torch.uint8)
    return whole[margin:margin + size], whole


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("kh,g,most", [(2, 4, 6), (1, 1, 2), (2, 8, 30)])
def test_captured_call_with_any_first_stays_inside(cuda, type_, kh, g, most):
    """Counts that a replay finds in device memory, the ends of 32 bits among them. 16 KB
    on both sides of workspace and outputs stay as they are, bit for bit, and a batch that
    is right after them gets its results."""
    torch = cuda
    new = [most, 1, 0, 2]
    b = shared.Batch(torch, kh, g, 64, 300, new, [most + 9, 1, 5, 60], type_, 9, ctx=96,
                     pad=(0, 4))
    sized = [between_margins(torch, n) for n in (b.size(), b.q.numel() * b.q.element_size())]
    b.work, b.att = sized[0][0], sized[1][0].view(b.q.dtype).view(b.q.shape)
    b.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    t = b.tokens
    for first in ([0, LOWEST, 0, 0, 0], [t - 3, LOWEST, t - 3, LOWEST, t],
                  [5, LOWEST + 5, 1, LOWEST + 1, 2], [HIGHEST, LOWEST, HIGHEST, LOWEST, HIGHEST],
                  [LOWEST, HIGHEST, LOWEST, HIGHEST, LOWEST], [0, HIGHEST, 3, HIGHEST - 1, t + 1],
                  [LOWEST, LOWEST + 1, LOWEST + 2, -1, HIGHEST], [0, 1 << 30, 5, 6, 7], b.first):
        b.d_first.copy_(torch.tensor(np.asarray(first).astype(np.int64), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for part, whole in sized:
            outside = whole.clone()
            at = part.data_ptr() - whole.data_ptr()
            outside[at:at + part.numel()] = 0x5A
            assert (outside == 0x5A).all(), first
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd,g,requests", [(32, 8, 300), (128, 8, 300), (64, 4, 520)])
def test_joins_of_many_rows(cuda, type_, hd, g, requests):
    """More rows of q heads than get a block each when their parts are joined."""
    b = shared.Batch(cuda, 2, g, hd, 70, [1] * requests, [1 + i % 40 for i in range(requests)],
                     type_, hd)
    assert requests * 2 * g > 4096
    b.run()
    b.check()
