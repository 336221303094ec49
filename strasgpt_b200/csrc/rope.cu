// strasgpt_k_rope: rotary positions given per token.
//
// Entry pair j of a head turns by the angle pos f_j (f_j: include/
// strasgpt_kernels.h):
//   (a, b) -> magnitude (a cos - b sin, a sin + b cos).
// The angle of a far position has no correct fp32 value (2^20 radians have
// an fp32 step of 1/8), so it is taken in turns and in 64 bits,
// pos (f_j / 2 pi), its whole turns are dropped exactly, and only the rest,
// at most half a turn, becomes an fp32 sine and cosine.
//
// What bounds it: bytes (each entry read and written once) for a chunk, one
// launch for a token. A block computes the sines of its tokens once, in
// shared memory, for all of its heads: their 64-bit part costs one multiply
// per pair and token instead of one per entry.
#include "entry.h"

#include <math.h>

extern "C" {
#include "strasgpt_kernels.h"
}

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;    // dim <= 512
constexpr int kUnroll = 4;        // items in flight per thread
constexpr int kSinesMax = 2048;   // (token, pair) sines of a block: 16 KB

struct RopeArgs {
  const void* x;
  void* y;
  long long xt, xh, yt, yh;  // token and head strides, in entries
  const int* pos;
  int t, heads, hd, dim;
  int tokens, heads_per_block;
  float magnitude;
  double turns[kMaxPairs];   // f_j / 2 pi
};

// V entries as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(uint16_t v) { return sg::bf16_to_f32(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
// Results are rounded once, to nearest even, as bf16 outputs are elsewhere.
__device__ __forceinline__ void from_f(float v, uint16_t& o) {
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(o) : "f"(v));
}

// An item is V pairs of one head (two accesses of V entries), or V entries
// behind the turned ones, which are copied.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) k_rope(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[kSinesMax];
  sg::pdl_trigger();
  sg::pdl_wait();
  const int half = a.dim / 2;
  const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.t - t0);
  const int h0 = blockIdx.y * a.heads_per_block, nh = min(a.heads_per_block, a.heads - h0);
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int token = i / half, j = i - token * half;
    const double turns = (double)a.pos[t0 + token] * a.turns[j];
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();

  const int turned = half / V, per_head = turned + (a.hd - a.dim) / V;
  const int items = nt * nh * per_head;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  using Access = Vec<T, V>;
  for (int i0 = threadIdx.x; i0 < items; i0 += kThreads * kUnroll) {
    Access p[kUnroll], q[kUnroll];
    long long to[kUnroll];
    int pair[kUnroll];  // index of the first pair's sine, or -1: copied
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      const int i = i0 + u * kThreads;
      if (i >= items) break;
      const int row = i / per_head, v = i - row * per_head;
      const int token = row / nh, h = h0 + row - token * nh;
      const long long from = (t0 + token) * a.xt + h * a.xh;
      to[u] = (t0 + token) * a.yt + h * a.yh;
      if (v < turned) {
        const int at = INTERLEAVED ? 2 * v * V : v * V;
        const int next = INTERLEAVED ? V : half;
        p[u] = *reinterpret_cast<const Access*>(x + from + at);
        q[u] = *reinterpret_cast<const Access*>(x + from + at + next);
        to[u] += at;
        pair[u] = token * half + v * V;
      } else {
        const int at = a.dim + (v - turned) * V;
        p[u] = *reinterpret_cast<const Access*>(x + from + at);
        to[u] += at;
        pair[u] = -1;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      if (i0 + u * kThreads >= items) break;
      if (pair[u] < 0) {
        *reinterpret_cast<Access*>(y + to[u]) = p[u];
        continue;
      }
      Access r, s;
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float2 k = cs[pair[u] + e];
        // Adjacent layout: the two accesses hold entries 0..V-1 and V..2V-1
        // of the run, and pair e is its entries 2e and 2e + 1.
        float f, g;
        if (INTERLEAVED) {
          f = to_f(2 * e < V ? p[u].e[2 * e % V] : q[u].e[2 * e % V]);
          g = to_f(2 * e + 1 < V ? p[u].e[(2 * e + 1) % V] : q[u].e[(2 * e + 1) % V]);
        } else {
          f = to_f(p[u].e[e]);
          g = to_f(q[u].e[e]);
        }
        const float n = f * k.x - g * k.y, m = f * k.y + g * k.x;
        if (INTERLEAVED) {
          from_f(n, 2 * e < V ? r.e[2 * e % V] : s.e[2 * e % V]);
          from_f(m, 2 * e + 1 < V ? r.e[(2 * e + 1) % V] : s.e[(2 * e + 1) % V]);
        } else {
          from_f(n, r.e[e]);
          from_f(m, s.e[e]);
        }
      }
      *reinterpret_cast<Access*>(y + to[u]) = r;
      *reinterpret_cast<Access*>(y + to[u] + (INTERLEAVED ? V : half)) = s;
    }
  }
}

template <typename T, int V>
cudaError_t launch(const RopeArgs& a, bool interleaved, dim3 grid, cudaStream_t s) {
  return interleaved ? sg::try_launch(k_rope<T, V, true>, grid, kThreads, 0, 1, s, a)
                     : sg::try_launch(k_rope<T, V, false>, grid, kThreads, 0, 1, s, a);
}

// Whether rows of `hd` entries at i st + j sh (i < t, j < heads) share no
// entry: one of the two strides steps over everything under the other.
bool rows_apart(long long t, long long st, long long heads, long long sh, long long hd) {
  if (st < 0 || sh < 0) return false;
  if ((t > 1 && st < hd) || (heads > 1 && sh < hd)) return false;
  if (t == 1 || heads == 1) return true;
  return st >= (heads - 1) * sh + hd || sh >= (t - 1) * st + hd;
}

}  // namespace

extern "C" int strasgpt_k_rope(const void* x, long long x_token_stride, long long x_head_stride,
                               void* y, long long y_token_stride, long long y_head_stride,
                               int type, int t, int heads, int head_dim, const int* pos,
                               const strasgpt_rope_t* rope, void* stream) {
  const char* const me = "strasgpt_k_rope";
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return sg::refuse(me, "unknown type");
  if (t < 0 || heads <= 0 || head_dim <= 0) return sg::refuse(me, "empty shape");
  if (heads > 65535 || head_dim > 65536) return sg::refuse(me, "too many heads or entries");
  if (!rope) return sg::refuse(me, "null parameters");
  if (rope->dim < 2 || rope->dim % 2 || rope->dim > head_dim || rope->dim > 2 * kMaxPairs)
    return sg::refuse(me, "the turned part must be even, 2 to min(head_dim, 512) entries");
  if (!(rope->theta > 0) || !isfinite(rope->theta)) return sg::refuse(me, "theta must be positive");
  if (!isfinite(rope->magnitude)) return sg::refuse(me, "magnitude must be finite");
  if (rope->scaling < STRASGPT_ROPE_NONE || rope->scaling > STRASGPT_ROPE_BANDS)
    return sg::refuse(me, "unknown scaling");
  if (rope->scaling != STRASGPT_ROPE_NONE && (!(rope->factor > 0) || !isfinite(rope->factor)))
    return sg::refuse(me, "factor must be positive");
  if (rope->scaling == STRASGPT_ROPE_BANDS &&
      (!(rope->low < rope->high) || !isfinite(rope->low) || !isfinite(rope->high) ||
       rope->original <= 0))
    return sg::refuse(me, "bands need low < high and a positive original length");
  if (t == 0) return 0;
  if (!x || !y || !pos) return sg::refuse(me, "null buffer");
  if (x_token_stride < 0 || x_head_stride < 0) return sg::refuse(me, "negative stride");
  if (!rows_apart(t, y_token_stride, heads, y_head_stride, head_dim))
    return sg::refuse(me, "rows of y overlap");
  if (x == y && ((t > 1 && x_token_stride != y_token_stride) ||
                 (heads > 1 && x_head_stride != y_head_stride)))
    return sg::refuse(me, "in place, x and y must have the same strides");
  const size_t size = type == STRASGPT_F32 ? 4 : 2;
  if (!sg::aligned(x, size) || !sg::aligned(y, size) || !sg::aligned(pos, 4))
    return sg::refuse(me, "a buffer is not aligned to its entries");
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {x, (const void*)y, (const void*)pos})
    if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);

  RopeArgs a;
  a.x = x; a.y = y; a.pos = pos;
  a.xt = x_token_stride; a.xh = x_head_stride;
  a.yt = y_token_stride; a.yh = y_head_stride;
  a.t = t; a.heads = heads; a.hd = head_dim; a.dim = rope->dim;
  a.magnitude = (float)rope->magnitude;
  const double two_pi = 6.283185307179586476925;
  const int half = rope->dim / 2;
  // f_j = theta^(-2 j / dim) as a running product: 255 roundings of 2^-53 at
  // most, far below what the fp32 sine keeps.
  const double ratio = pow(rope->theta, -2.0 / rope->dim);
  double f = 1.0;
  for (int j = 0; j < half; j++, f *= ratio) {
    double g = f;
    if (rope->scaling == STRASGPT_ROPE_LINEAR) {
      g = f / rope->factor;
    } else if (rope->scaling == STRASGPT_ROPE_BANDS) {
      const double turns = rope->original * f / two_pi;
      double keep = (turns - rope->low) / (rope->high - rope->low);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      g = f * (keep + (1 - keep) / rope->factor);
    }
    a.turns[j] = g / two_pi;
  }

  // 16-byte accesses where every run of V entries starts on 16 bytes, single
  // entries otherwise.
  const int wide = (int)(16 / size);
  const bool vec = half % wide == 0 && (head_dim - rope->dim) % wide == 0 &&
                   a.xt % wide == 0 && a.xh % wide == 0 && a.yt % wide == 0 &&
                   a.yh % wide == 0 && sg::aligned(x, 16) && sg::aligned(y, 16);
  const int v = vec ? wide : 1;
  const int per_head = half / v + (head_dim - rope->dim) / v;
  // Blocks of one item per thread while they all fit on the GPU at once
  // (8 blocks per SM), of kUnroll items per thread after that.
  const long long all = (long long)t * heads * per_head;
  const int target = all <= (long long)sms * 8 * kThreads ? kThreads : kThreads * kUnroll;
  a.heads_per_block = (target + per_head - 1) / per_head;
  if (a.heads_per_block > heads) a.heads_per_block = heads;
  a.tokens = target / (a.heads_per_block * per_head);
  if (a.tokens > kSinesMax / half) a.tokens = kSinesMax / half;
  if (a.tokens > t) a.tokens = t;
  if (a.tokens < 1) a.tokens = 1;
  const dim3 grid((t + a.tokens - 1) / a.tokens,
                  (heads + a.heads_per_block - 1) / a.heads_per_block);
  const bool il = rope->interleaved != 0;
  const cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (type == STRASGPT_F32)
    e = vec ? launch<float, 4>(a, il, grid, s) : launch<float, 1>(a, il, grid, s);
  else
    e = vec ? launch<uint16_t, 8>(a, il, grid, s) : launch<uint16_t, 1>(a, il, grid, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}
