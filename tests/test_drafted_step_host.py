"""Host side of the entry points of a step over drafted tokens, compiled from
its sources into small programs that need no GPU: calls into the CUDA runtime
are replaced by ones that the program defines.
"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_program(tmp_path, source):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "program.cu", tmp_path / "program"
    src.write_text(source)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1",
                    f"-I{ROOT}/include", f"-I{ROOT}/strasgpt_b200/csrc", "-o", str(exe), str(src)],
                   check=True, timeout=600)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr


def test_shared_memory_limit_is_never_lowered(tmp_path):
    """Two threads' first calls with different sizes: the larger one's limit is
    set first, the smaller one's call comes before it is noted. What is noted
    then is what the kernel has."""
    run_program(tmp_path, r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<int> limit{0}, large_set{0}, small_returned{0};
template <typename F>
static void wait_for(F ready) {   // half a second at most
  for (int i = 0; i < 500 && !ready(); i++)
    std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
template <typename K>
static cudaError_t fake_set(K, cudaFuncAttribute, int bytes) {
  limit = bytes;
  if (bytes == 200000) {
    large_set = 1;
    wait_for([] { return small_returned == 1; });
  }
  return cudaSuccess;
}
#define cudaFuncSetAttribute fake_set
#include "entry.h"
static void kernel() {}
int main() {
  static std::atomic<size_t> done[sg::kDevices];
  std::thread a([] { sg::allow_smem(&kernel, 200000, 3, done); });
  std::thread b([] {
    wait_for([] { return large_set == 1; });
    sg::allow_smem(&kernel, 100000, 3, done);
    small_returned = 1;
  });
  a.join();
  b.join();
  printf("limit %d, noted %zu\n", (int)limit, (size_t)done[3]);
  if (limit != 200000 || done[3] != 200000) return 1;
  // A larger size raises it, a smaller one does nothing, other devices have
  // limits of their own.
  sg::allow_smem(&kernel, 210000, 3, done);
  sg::allow_smem(&kernel, 1000, 3, done);
  if (limit != 210000 || done[3] != 210000 || done[2] != 0) return 2;
  return 0;
}
""")


def test_last_fill_of_a_stage_is_waited_for(tmp_path):
    """A barrier's wait on a parity ends when the phase that is under way has
    the other one. For every number of tiles and stages the wait for a stage's
    last fill lasts while that fill is on its way, and ends once it has landed."""
    run_program(tmp_path, r"""
#include "attn_tree.h"
#include <cstdio>
int main() {
  for (int stages = 1; stages <= 8; stages++)
    for (int asked = 1; asked <= 5 * stages + 3; asked++)
      for (int s = 0; s < stages && s < asked; s++) {
        int fills = 0;
        for (int i = s; i < asked; i += stages) fills++;
        const unsigned parity = sg::tree_last_parity(asked, s, stages);
        for (int landed = fills - 1; landed <= fills; landed++) {
          const unsigned under_way = (unsigned)landed & 1;   // phases count from 0
          const bool ends = under_way != parity;
          if (ends != (landed == fills)) {
            printf("%d stages, %d tiles, stage %d: %d of %d landed, wait %s\n", stages, asked, s,
                   landed, fills, ends ? "ends" : "lasts");
            return 1;
          }
        }
      }
  return 0;
}
""")
