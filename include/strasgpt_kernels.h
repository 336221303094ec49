// strasgpt-b200 kernel-level entry points, for unit tests and for callers
// that manage their own device buffers. All pointers are DEVICE pointers;
// `stream` is a cudaStream_t (NULL: the legacy default stream). Each call
// only enqueues work; it returns 0, or dies with "[StrasGPT] Error ..." on an
// invalid shape (or, where it says so, returns -1). None of these has a
// counterpart in the reference API: they expose the pieces of
// transformer_predict_chunk (source/transformer.c:1186-1602) one at a time.
#ifndef STRASGPT_KERNELS_H
#define STRASGPT_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// Epilogue selector shared by the projection entry points.
#define STRASGPT_EPI_STORE  0  // out = W x
#define STRASGPT_EPI_ADD    1  // out += W x (residual)
#define STRASGPT_EPI_SWIGLU 2  // out = silu(gate) * up, gate/up rows interleaved

// y = W x for one token: W bf16 [rows][K] (rows of K contiguous), x fp32
// [K]. norm_w (bf16 [K]) != NULL applies the reference RMSNorm to x first
// (source/transformer.c:978-999). For STRASGPT_EPI_SWIGLU `rows` counts
// outputs and W holds 2*rows rows: gate row f at 2f, up row f at 2f+1.
int strasgpt_k_matvec(const float* x, const uint16_t* norm_w, float eps,
                      const uint16_t* w, int k, int rows, float* out, int epi,
                      void* stream);

// C[m][n] (op)= sum_k A[m][k] W[n][k] for m < M, n < N (SIMT fp32 tiles).
// For STRASGPT_EPI_SWIGLU, N counts weight rows and C has N/2 columns.
int strasgpt_k_gemm_simt(const float* a, int lda, const uint16_t* w, int k,
                         int m, int n, float* c, int ldc, int epi,
                         void* stream);

// Same product as strasgpt_k_gemm_simt on the tcgen05 tensor cores: A is
// split into bf16 halves a_hi + a_lo (caller-provided [m][k] buffers,
// 16-byte aligned, k a multiple of 8) and both are multiplied with W in fp32
// accumulation. `err` is a device int, zero at rest, set non-zero if the
// kernel's pipeline waits time out (C is then incomplete).
int strasgpt_k_gemm_tc(const float* a, int lda, uint16_t* a_hi,
                       uint16_t* a_lo, const uint16_t* w, int k, int m, int n,
                       float* c, int ldc, int epi, int* err, void* stream);

// Causal GQA attention of a chunk (source/transformer.c:1375-1422): q
// [t][kv_heads*group][head_dim] at positions pos0.., caches
// [kv_heads][ctx][head_dim] holding keys/values 0..pos0+t-1; att gets
// [t][kv_heads*group][head_dim]. head_dim 32, 64 or 128; group divides 64.
int strasgpt_k_attn_prefill(const float* q, const float* k_cache,
                            const float* v_cache, int t, int kv_heads,
                            int group, int head_dim, int ctx, int pos0,
                            float* att, void* stream);

// y[t] = rmsnorm(x[t]) * w for t < T, rows of D floats.
int strasgpt_k_rmsnorm_rows(const float* x, int t, int d, const uint16_t* w,
                            float eps, float* y, void* stream);

// The error path of the device-side waits, for tests (no counterpart in the
// reference): runs the tensor-parallel barrier kernel of a 2-rank exchange
// on the current GPU whose second rank is a buffer that nothing writes
// (peer_posted 0: the wait can only run out) or whose post is already in
// place (peer_posted 1), with a wait limit of timeout_ms. Returns 1 when
// the wait ran out and the kernel returned with its error flag set, 0 when
// it completed, -1 on a bad argument. The GPU stays usable either way.
int strasgpt_k_tp_wait_check(int timeout_ms, int peer_posted, void* stream);

// Size of the fixed device scratch of strasgpt_k_matvec_noalloc, held by
// every GPU that loads the library until the process exits.
#define STRASGPT_NOALLOC_SCRATCH_BYTES (4 << 20)

// strasgpt_k_matvec without any allocation, for callers that own all of the
// GPU's memory through their own pools or cannot stall the device with
// cudaMalloc/cudaFree between decode steps. No counterpart in the reference:
// it is an extra way in to the same projection. Same arguments and result as
// strasgpt_k_matvec (computed split-K: fp32 sums in another order); x, w and
// norm_w must be 16-byte aligned. Its scratch is a fixed 4 MiB device array:
// the weight rows (2*rows for STRASGPT_EPI_SWIGLU) may be at most
// STRASGPT_NOALLOC_SCRATCH_BYTES / 4 - 64 = 1048512; larger shapes, and
// other invalid arguments, return -1 with a message on stderr and enqueue
// nothing. The first call on a device looks up the scratch's address, so
// make it before any stream capture on that device. All calls on a device
// share the scratch: calls that overlap on the GPU race, so serialise them
// (one stream). Returns 0 once the work is enqueued.
int strasgpt_k_matvec_noalloc(const float* x, const uint16_t* norm_w,
                              float eps, const uint16_t* w, int k, int rows,
                              float* out, int epi, void* stream);

// --- A step over drafted tokens --------------------------------------------
// The three entry points below have no counterpart in the reference. They
// read a drafted tree of tokens: rotate its queries and keys, attend over the
// cache and the tree, choose a token from each row of logits. Buffers are
// device memory of the current device; `type` is STRASGPT_F32 (float) or
// STRASGPT_BF16 (uint16_t) for every buffer given as void*; strides count
// entries. They allocate nothing, keep nothing between calls, and can be
// captured into a CUDA graph, which keeps the addresses and numbers of the
// call and reads what is in device memory (positions, lengths, masks, filters,
// random numbers) at each replay. Each returns 0 once its work is enqueued; an
// invalid argument or a buffer that is not on the current device returns -1
// with a "[StrasGPT] Error ..." message on stderr and enqueues nothing. A
// launch that fails returns -1 with a message too; attention and sampling may
// be two launches, of which the first is then enqueued: outputs and workspace
// hold nothing of use. What is in device memory cannot be refused: each says
// what it does with any value.
#define STRASGPT_F32  0
#define STRASGPT_BF16 1

// How far entry pair j (j < dim / 2) of a head turns per position, in
// radians, with f = theta^(-2 j / dim):
//   STRASGPT_ROPE_NONE    f
//   STRASGPT_ROPE_LINEAR  f / factor
//   STRASGPT_ROPE_BANDS   f (k + (1 - k) / factor), where k goes from 0 to 1
//                         as the turns that f makes over `original`
//                         positions, original f / (2 pi), go from low to high:
//                         short wavelengths keep their frequency, long ones
//                         are stretched by factor
#define STRASGPT_ROPE_NONE   0
#define STRASGPT_ROPE_LINEAR 1
#define STRASGPT_ROPE_BANDS  2
typedef struct strasgpt_rope {
  int dim;          // entries that turn, the first of the head: even, 2..512
  int interleaved;  // pairs (2j, 2j + 1); 0: pairs (j, j + dim / 2)
  int scaling;      // STRASGPT_ROPE_*
  int original;     // BANDS: positions of the unstretched context
  double theta;     // > 0
  double factor;    // LINEAR, BANDS: > 0
  double low, high; // BANDS: low < high
  double magnitude; // the turned entries are multiplied by it (1: as they are)
} strasgpt_rope_t;

// Rotary positions: row (i, h), i < t, h < heads, of head_dim entries at
// x + i * x_token_stride + h * x_head_stride is turned by its angles at
// position pos[i] (any int: tokens may share a position, a negative one turns
// back) and written to y + i * y_token_stride + h * y_head_stride; entries
// behind the first rope->dim are copied. Angles are computed in 64 bits, the
// rest in 32 (frequencies of 1e298 turns and more are refused). y is x with the
// same strides (in place), or shares no memory with x's rows; rows of y must
// not overlap. With the strides of a layer's cache ([kv_heads][ctx][head_dim]:
// head_dim and ctx * head_dim) it appends keys. y is an address: a captured call writes the same cache rows at every
// replay. Where a graph is to serve other lengths, as strasgpt_k_attn_tree's
// does, let it write to a buffer and copy the rows into the cache outside the
// graph (or capture again, or update the node). t 0 does nothing.
int strasgpt_k_rope(const void* x, long long x_token_stride,
                    long long x_head_stride, void* y, long long y_token_stride,
                    long long y_head_stride, int type, int t, int heads,
                    int head_dim, const int* pos, const strasgpt_rope_t* rope,
                    void* stream);

// GQA attention of t drafted tokens (at most STRASGPT_ATTN_TREE_MAX) over a
// cache. q holds token i's kv_heads * group heads of head_dim entries at
// q + i * ldq, att gets the outputs at att + i * ldo in the same order; the
// caches are [kv_heads][ctx][head_dim] as in strasgpt_k_attn_prefill. Rows
// 0..*cached - 1 of the caches are seen by every token, rows *cached + j are
// the drafted tokens' own: token i sees j where bit j % 64 of
// mask[i * ((t + 63) / 64) + j / 64] is set (its own bit included, or it does
// not see itself). Scores are q.k / sqrt(head_dim); sums and maxima are held
// in 32 bits. Products keep 21 bits of each fp32 operand at least; bf16 ones
// are exact, the probabilities that multiply bf16 values keep 17 bits. A token
// that sees nothing gets zeros.
//
// Rows that a token does not see, and rows behind the last, may hold anything
// (infinities and NaN too). Rows that it sees hold finite numbers: an infinity
// or NaN among them leaves that token's outputs of the q heads on that kv head
// unspecified (infinite, NaN, or as if the row were not there, by the number of
// rows), and no others. att is q with ldo = ldq (in place), or shares no memory
// with what is read. *cached is read on the device and cut to 0..ctx - t.
// head_dim 32, 64 or 128; group 1..128; q, the caches, att, their rows and the
// workspace are 16-byte aligned.
//
// The workspace has strasgpt_k_attn_tree_workspace(t, kv_heads, group,
// head_dim) bytes (asked on the same device; 0: may be NULL). Its contents
// matter only during a call; calls that may overlap on the GPU, replays of
// two captured graphs among them, need one each.
#define STRASGPT_ATTN_TREE_MAX 1024
size_t strasgpt_k_attn_tree_workspace(int t, int kv_heads, int group,
                                      int head_dim);
int strasgpt_k_attn_tree(const void* q, long long ldq, const void* k_cache,
                         const void* v_cache, int type, int t, int kv_heads,
                         int group, int head_dim, int ctx, const int* cached,
                         const uint64_t* mask, void* att, long long ldo,
                         void* workspace, size_t workspace_bytes, void* stream);

// One token for each row of logits (rows of vocab entries, ld apart), from
// the row's random number u in [0, 1). Per row, NULL for none:
//   temperature  w = exp((x - max x) / temperature); 1 if NULL; the largest
//                logit (lowest index among equals) if not above 0
//   top_k        the k largest stay; all if not above 0
//   top_p        then the fewest, largest first, whose mass reaches top_p of
//                what top_k left; all if not below 1, the largest if not
//                above 0
//   min_p        then those with w >= min_p (1 at most); all if not above 0
// Equal logits rank by index, lowest first. The token is the first remaining
// one, in index order, at which the running sum of w exceeds u times the sum
// of all that remain (u not above 0: the first, u not below 1: the last; an
// entry whose w is 0 in 64 bits is never drawn). Weights and sums are held in
// 64 bits, weights to 2^-42 of themselves; where top_p's border, or the mass
// of what the filters leave, is summed over a whole row, to 2^-30, which counts
// where a border lies that close to an entry's end. prob (NULL: not wanted)
// gets the token's share of the remaining mass, kept (NULL) how many entries
// remained. NaN logits count as -inf, which are never taken; a row of nothing
// else gets token -1, prob 0, kept 0. Where logits are +inf, those weigh 1 and
// all others 0. vocab is at most STRASGPT_SAMPLE_MAX_VOCAB. token, prob and
// kept share no memory with each other or the inputs. The result does not
// depend on timing: the same inputs give the same bits.
#define STRASGPT_SAMPLE_MAX_VOCAB 360448
int strasgpt_k_sample(const void* logits, int type, long long ld, int rows,
                      int vocab, const float* temperature, const int* top_k,
                      const float* top_p, const float* min_p, const float* u,
                      int* token, float* prob, int* kept, void* stream);

#ifdef __cplusplus
}
#endif

#endif // STRASGPT_KERNELS_H
