// What the two kernels behind strasgpt_k_attn_tree share: attn_tree.cu (the
// entry point, few rows per kv head) and attn_tree_tc.cu (many).
#pragma once

#include "entry.h"

namespace sg {

struct TreeArgs {
  const void* q;
  const void* k;
  const void* v;
  void* att;
  long long ldq, ldo;
  int t, kh, group, ctx, words;
  const int* cached;
  const unsigned long long* mask;
  int splits;
  float* part;     // [splits][kh][t * group][HD] outputs before division
  float2* ml;      // [splits][kh][t * group] running maximum (base 2) and sum
};

// Cached keys, cut to what the cache holds.
__device__ __forceinline__ int tree_cached(const TreeArgs& a) {
  return min(max(*a.cached, 0), a.ctx - a.t);
}

// The cached keys [0, *cached) on the fifth-generation tensor cores, 128 rows
// per CTA; the drafted ones are k_merge's. head_dim 64 or 128.
constexpr int kTreeTcRows = 128;
cudaError_t tree_tc(const TreeArgs& a, bool f32, int head_dim, int dev, cudaStream_t s);
// Keys per tile: what a split's share is a multiple of.
int tree_tc_keys();

// Tiles i = 0, 1, ... go to a ring of `stages`, tile i to stage i % stages, and
// each fill of a stage completes a phase of its barrier. The parity of the
// phase that stage s's last fill completes, when `asked` > s tiles were asked
// for: a wait on it ends when that fill has landed, and not at an older one.
__host__ __device__ constexpr unsigned tree_last_parity(int asked, int s, int stages) {
  return (unsigned)((asked - 1 - s) / stages) & 1u;
}

}  // namespace sg
