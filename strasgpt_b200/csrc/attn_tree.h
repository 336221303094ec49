// What the kernels behind strasgpt_k_attn_tree and strasgpt_k_attn_shared share:
// attn_tree.cu (the entry points, few rows per kv head) and attn_tree_tc.cu
// (many).
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
  int drafted;     // keys behind the cached ones that the mask is about: t, or 0
  const int* cached;
  const unsigned long long* mask;
  int splits;
  float* part;     // [splits][kh][t * group][HD] outputs before division
  float2* ml;      // [splits][kh][t * group] running maximum (base 2) and sum
  bool whole;      // one split writes att; else, and always where not set, parts
};

// Cached keys, cut to what the cache holds.
__device__ __forceinline__ int tree_cached(const TreeArgs& a) {
  return min(max(*a.cached, 0), a.ctx - a.drafted);
}

// Rows from..to - 1 of a call with `tokens` rows, as far as they are there and `most`
// of them at most: the first one and how many. Any from and to, which device memory
// holds, give rows of the call, or none: both ends are cut before they are subtracted.
__host__ __device__ inline void cut_tokens(long long from, long long to, int tokens, int most,
                                           int* token0, int* count) {
  const int begin = (int)(from < 0 ? 0 : from > tokens ? tokens : from);
  const int end = (int)(to < 0 ? 0 : to > tokens ? tokens : to);
  *token0 = begin;
  *count = end <= begin ? 0 : end - begin < most ? end - begin : most;
}

// A batch of requests whose t tokens are in all, each request's next to one
// another: k, v and ctx are the requests' own caches', and a request's tokens
// see each other in order.
struct BatchArgs : TreeArgs {
  int requests, most;        // most: of a request's tokens
  const int* first;          // [requests + 1], or NULL: most each
  const int* rows;           // [requests]: of its cache, its tokens' included
  long long stride;          // entries from one request's cache to the next's
  int ctas;                  // that share the requests' tiles
  int split0;                // parts of the prefix come before the requests' own
  int2* where;               // [kh][t * group]: which CTAs a row's own parts are of
};

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
