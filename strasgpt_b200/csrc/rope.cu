// strasgpt_k_rope, strasgpt_k_rope_axes: rotary positions given per token, or
// per token and axis.
//
// Entry pair j of a head turns by the angle pos f_j (f_j: include/
// strasgpt_kernels.h):
//   (a, b) -> magnitude (a cos - b sin, a sin + b cos).
// The angle of a far position has no correct fp32 value (2^20 radians have
// an fp32 step of 1/8), so it is taken in turns and in 64 bits,
// pos (f_j / 2 pi), its whole turns are dropped exactly, and the rest, at most
// half a turn, is an fp32 angle, whose sine and cosine fp32 computes, plus
// (fp32 rows) what its rounding left, less than 2^-23, to first order. That
// correction and the magnitude, as two fp32 values, come to one rounding.
//
// What bounds it: bytes (each entry read and written once) for a chunk of fp32,
// instruction issue (73 % of cycles) for one of bf16, one launch for a token.
// A block has a run of items (two a thread), loads them first, and computes
// the sines of their tokens, once for all heads, in shared memory while they
// are on their way: the sines' 64-bit part costs a multiply per pair and token
// instead of one per entry. Measured on a B200:
// 1.8 us for one token of 40 heads of 128 fp32 entries, 4.5 us (3.7 TB/s) for
// 2048 tokens of 8 such heads into a cache, 44 us (3.8 TB/s; a plain copy of
// as many contiguous bytes takes 33) for 8191 tokens of 40 heads of 128 bf16
// entries, half of each turned, out of rows twice as wide. On several axes: 2.1 us for
// one token of 40 heads of 128 fp32 entries, 5.4 us for 2048 tokens of 8 such heads
// into a cache, 23.5 us (3.6 TB/s) for 8191 tokens of 32 heads of 80 bf16 entries.
#include "entry.h"

#include <limits.h>
#include <math.h>

extern "C" {
#include "strasgpt_kernels.h"
}

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;    // dim <= 512
constexpr int kUnroll = 2;        // items in flight per thread
constexpr int kSinesMax = 2048;   // (token, pair) sines of a block: 16 KB

// Division of numbers below 2^31 by d, 1..2^30, as a product: with 2^(b - 1) < d <=
// 2^b and mul = floor(2^(31 + b) / d) + 1, mul d is above 2^(31 + b) by 2^b at most,
// which n < 2^31 does not carry into the quotient. (A division by a number that is
// not known beforehand takes some 30 instructions, three of them an item, where
// instructions are what counts: 8191 tokens of 32 heads of 80 bf16 entries 23.9 ->
// 23.5 us.)
struct Divisor {
  unsigned d, mul, shift;
  Divisor() = default;
  explicit Divisor(unsigned by) : d(by) {
    unsigned b = 0;
    while ((1u << b) < by) b++;
    mul = (unsigned)((1ull << (31 + b)) / by + 1);
    shift = b - 1;  // (by 1: not used)
  }
};
__device__ __forceinline__ int divide(int n, const Divisor& by) {
  return by.d == 1 ? n : (int)(__umulhi((unsigned)n, by.mul) >> by.shift);
}

struct RopeArgs {
  const void* x;
  void* y;
  long long xt, xh, yt, yh;  // token and head strides, in entries
  const int* pos;
  int t, heads, hd, dim;
  int per_block;             // items of a block
  Divisor token_items, head_items, token_pairs;  // items of a token, of a head; pairs
  float magnitude, magnitude_rest;  // their sum, to 48 bits
  double turns[kMaxPairs];   // f_j / 2 pi
};

// Several axes: pair j turns by the position of its axis.
struct AxesArgs : RopeArgs {
  long long pa, pt;          // axis and token strides of pos
  uint8_t axis[kMaxPairs];
};

// Position that turns pair j of a token.
__device__ __forceinline__ int position(const RopeArgs& a, int token, int) { return a.pos[token]; }
__device__ __forceinline__ int position(const AxesArgs& a, int token, int j) {
  return a.pos[a.axis[j] * a.pa + token * a.pt];
}

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

// How the pairs of a head are read.
enum Layout {
  kHalves,    // (j, j + dim / 2): V pairs are two accesses of V entries
  kAdjacent,  // (2j, 2j + 1): V / 2 pairs are one access (V >= 2)
  kSingle     // (2j, 2j + 1), entry by entry (V == 1)
};

// Blocks per SM that the registers are held to: two accesses an item need 64
// a thread (4 blocks; at 6 they spill, 22 us for 17 us on 4096 x 32 x 128 bf16
// entries), one gets by with 40 (6; 44 us for 55 us on 8191 x 40 x 128).
constexpr int blocks_of(Layout l) { return l == kHalves ? 4 : 6; }

// An item is the pairs of one access, or V entries behind the turned ones,
// which are copied.
template <typename T, int V, Layout LAYOUT, typename Args>
__global__ void __launch_bounds__(kThreads, blocks_of(LAYOUT))
    k_rope(const __grid_constant__ Args a) {
  constexpr int kPairs = LAYOUT == kAdjacent ? V / 2 : V;  // of an item
  constexpr bool kTwo = LAYOUT != kAdjacent;               // two accesses
  __shared__ float2 cs[kSinesMax];
  const int half = a.dim / 2, next = LAYOUT == kSingle ? 1 : half;
  // Items in the order token, head, place: a block has a run of them, of
  // tokens t0 to t0 + nt - 1, and starts at place `skip` of the first.
  const int turned = half / kPairs, per_head = turned + (a.hd - a.dim) / V;
  const int per_token = a.heads * per_head;
  const long long first = (long long)blockIdx.x * a.per_block, all = (long long)a.t * per_token;
  const int t0 = (int)(first / per_token), skip = (int)(first - (long long)t0 * per_token);
  const int items = (int)min((long long)a.per_block, all - first);
  const int nt = (skip + items - 1) / per_token + 1;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  using Access = Vec<T, V>;
  Access p[kUnroll], q[kTwo ? kUnroll : 1];
  long long to[kUnroll];
  int pair[kUnroll];  // where the item's sines are, or -1: copied
  sg::pdl_trigger();
  sg::pdl_wait();
  // The entries are on their way while the sines are computed.
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const int i = threadIdx.x + u * kThreads;
    if (i >= items) break;
    const int token = divide(skip + i, a.token_items), place = skip + i - token * per_token;
    const int h = divide(place, a.head_items), v = place - h * per_head;
    const bool turn = v < turned;
    const int at = !turn ? a.dim + (v - turned) * V : LAYOUT == kSingle ? 2 * v : v * V;
    const T* from = x + (t0 + token) * a.xt + h * a.xh + at;
    p[u] = *reinterpret_cast<const Access*>(from);
    if (kTwo && turn) q[kTwo ? u : 0] = *reinterpret_cast<const Access*>(from + next);
    to[u] = (t0 + token) * a.yt + h * a.yh + at;
    pair[u] = turn ? token * half + v : -1;
  }
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int token = divide(i, a.token_pairs), j = i - token * half;
    const double turns = (double)position(a, t0 + token, j) * a.turns[j];
    const double half_turns = 2.0 * (turns - rint(turns));
    const float near = (float)half_turns;
    float s, c, s_rest = 0.f, c_rest = 0.f;
    sincospif(near, &s, &c);
    // (A bf16 result would not show it; 8191 tokens of 40 heads 43.7 -> 44.7 us.)
    if constexpr (sizeof(T) == 4) {
      const float rest = (float)(half_turns - near) * 3.14159265f * a.magnitude;
      s_rest = fmaf(s, a.magnitude_rest, c * rest);
      c_rest = fmaf(c, a.magnitude_rest, -s * rest);
    }
    // Pair kPairs v + e of a token lies at e turned + v: the sines of an item
    // are read by neighbouring threads side by side.
    cs[token * half + j % kPairs * turned + j / kPairs] =
        make_float2(fmaf(c, a.magnitude, c_rest), fmaf(s, a.magnitude, s_rest));
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    if (threadIdx.x + u * kThreads >= items) break;
    if (pair[u] >= 0) {
#pragma unroll
      for (int e = 0; e < kPairs; e++) {
        const float2 k = cs[pair[u] + e * turned];
        T& one = kTwo ? p[u].e[e] : p[u].e[2 * e % V];
        T& two = kTwo ? q[kTwo ? u : 0].e[e] : p[u].e[(2 * e + 1) % V];
        const float f = to_f(one), g = to_f(two);
        from_f(f * k.x - g * k.y, one);
        from_f(f * k.y + g * k.x, two);
      }
      if (kTwo) *reinterpret_cast<Access*>(y + to[u] + next) = q[kTwo ? u : 0];
    }
    *reinterpret_cast<Access*>(y + to[u]) = p[u];
  }
}

template <typename T, int V, typename Args>
cudaError_t launch(const Args& a, bool interleaved, dim3 grid, cudaStream_t s) {
  constexpr Layout kPaired = V > 1 ? kAdjacent : kSingle;
  return interleaved ? sg::try_launch(k_rope<T, V, kPaired, Args>, grid, kThreads, 0, 1, s, a)
                     : sg::try_launch(k_rope<T, V, kHalves, Args>, grid, kThreads, 0, 1, s, a);
}

// Whether rows of `hd` entries at i st + j sh (i < t, j < heads) share no
// entry: one of the two strides steps over everything under the other.
bool rows_apart(long long t, long long st, long long heads, long long sh, long long hd) {
  if (st < 0 || sh < 0) return false;
  if ((t > 1 && st < hd) || (heads > 1 && sh < hd)) return false;
  if (t == 1 || heads == 1) return true;
  return st >= (heads - 1) * sh + hd || sh >= (t - 1) * st + hd;
}

// Why the parameters are refused, or NULL.
const char* bad_parameters(const strasgpt_rope_t* rope, int head_dim) {
  if (!rope) return "null parameters";
  if (rope->dim < 2 || rope->dim % 2 || rope->dim > head_dim || rope->dim > 2 * kMaxPairs)
    return "the turned part must be even, 2 to min(head_dim, 512) entries";
  if (!(rope->theta > 0) || !isfinite(rope->theta)) return "theta must be positive";
  if (!isfinite((float)rope->magnitude)) return "magnitude must be finite";
  if (rope->scaling < STRASGPT_ROPE_NONE || rope->scaling > STRASGPT_ROPE_BANDS)
    return "unknown scaling";
  if (rope->scaling != STRASGPT_ROPE_NONE && (!(rope->factor > 0) || !isfinite(rope->factor)))
    return "factor must be positive";
  if (rope->scaling == STRASGPT_ROPE_BANDS &&
      (!(rope->low < rope->high) || !isfinite(rope->low) || !isfinite(rope->high) ||
       rope->original <= 0))
    return "bands need low < high and a positive original length";
  return nullptr;
}

// Turns per position of `count` pairs, f_m = theta^(-m / count), m = 0, 1, ...,
// to turns[at(m)], and whether all of them, times any position, stay within 64
// bits.
//
// f_m is a running product in 64-bit mantissas: at most 255 roundings of 2^-64
// and as many times the ratio's own (2^-63), 2^-54 in all, so that a pair's
// turns per position are off by little more than their last rounding to 64
// bits (2^-53), which is what counts at far positions. (In doubles the product
// was off by up to 2^-46: 4e-6 radians at position 2^31 for 512 entries and
// theta 2.)
template <typename At>
bool turns_of(const strasgpt_rope_t& rope, int count, double* turns, At at) {
  const long double per_turn = 1 / 6.283185307179586476925286766559L;
  const long double ratio = powl(rope.theta, -2.0L / (2 * count));
  const long double stretched =
      rope.scaling == STRASGPT_ROPE_NONE ? per_turn : per_turn / rope.factor;
  long double f = 1;
  for (int m = 0; m < count; m++, f *= ratio) {
    long double t = stretched;
    if (rope.scaling == STRASGPT_ROPE_BANDS) {
      long double keep = (rope.original * f * per_turn - rope.low) /
                         ((long double)rope.high - rope.low);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      t = keep * per_turn + (1 - keep) * stretched;
    }
    turns[at(m)] = (double)(f * t);
    if (!(fabs(turns[at(m)]) < 1e298)) return false;
  }
  return true;
}

// Both entry points: checks, and the launch for arguments `a` whose positions
// and frequencies are set by `fill(a)` (which says why it refuses, or NULL).
template <typename Args, typename Fill>
int turn(const char* me, const void* x, long long x_token_stride, long long x_head_stride, void* y,
         long long y_token_stride, long long y_head_stride, int type, int t, int heads,
         int head_dim, const int* pos, const strasgpt_rope_t* rope, void* stream, Fill fill) {
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return sg::refuse(me, "unknown type");
  if (t < 0 || heads <= 0 || head_dim <= 0) return sg::refuse(me, "empty shape");
  if (heads > 65535 || head_dim > 65536) return sg::refuse(me, "too many heads or entries");
  if (const char* why = bad_parameters(rope, head_dim)) return sg::refuse(me, why);
  Args a;
  const char* const why_not = fill(a);
  if (t == 0) return why_not ? sg::refuse(me, why_not) : 0;
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
  if (why_not) return sg::refuse(me, why_not);
  a.x = x; a.y = y; a.pos = pos;
  a.xt = x_token_stride; a.xh = x_head_stride;
  a.yt = y_token_stride; a.yh = y_head_stride;
  a.t = t; a.heads = heads; a.hd = head_dim; a.dim = rope->dim;
  a.magnitude = (float)rope->magnitude;
  a.magnitude_rest = (float)(rope->magnitude - a.magnitude);
  const int half = rope->dim / 2;
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {x, (const void*)y, (const void*)pos})
    if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);

  // 16-byte accesses where every run of their entries starts on 16 bytes; for
  // adjacent pairs, else, an access per pair where pairs start on their size;
  // single entries otherwise.
  const bool il = rope->interleaved != 0;
  auto fits = [&](int v, int unit) {
    return unit % v == 0 && (head_dim - rope->dim) % v == 0 && a.xt % v == 0 && a.xh % v == 0 &&
           a.yt % v == 0 && a.yh % v == 0 && sg::aligned(x, v * size) && sg::aligned(y, v * size);
  };
  const int wide = (int)(16 / size), unit = il ? rope->dim : half;
  const int v = fits(wide, unit) ? wide : il && fits(2, unit) ? 2 : 1;
  const int per_head = (il && v > 1 ? rope->dim : half) / v + (head_dim - rope->dim) / v;
  // Blocks of one item per thread while they all fit on the GPU at once
  // (8 blocks per SM), of kUnroll after that; no more tokens than have room
  // for their sines (a block's run may start and end within a token).
  const long long per_token = (long long)heads * per_head, all = t * per_token;
  long long per_block = all <= (long long)sms * 8 * kThreads ? kThreads : kThreads * kUnroll;
  const long long room = (kSinesMax / half - 2) * per_token;
  a.per_block = (int)(room < per_block ? room : per_block);
  const long long blocks = (all + a.per_block - 1) / a.per_block;
  if (per_token > 1 << 30 || blocks > INT_MAX) return sg::refuse(me, "too many entries");
  a.token_items = Divisor((unsigned)per_token);
  a.head_items = Divisor((unsigned)per_head);
  a.token_pairs = Divisor((unsigned)half);
  const dim3 grid((unsigned)blocks);
  const cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (type == STRASGPT_F32)
    e = v == 4   ? launch<float, 4>(a, il, grid, s)
        : v == 2 ? launch<float, 2>(a, true, grid, s)
                 : launch<float, 1>(a, il, grid, s);
  else
    e = v == 8   ? launch<uint16_t, 8>(a, il, grid, s)
        : v == 2 ? launch<uint16_t, 2>(a, true, grid, s)
                 : launch<uint16_t, 1>(a, il, grid, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}

const char* const kTooFast = "frequencies beyond 64 bits";

}  // namespace

extern "C" {

int strasgpt_k_rope(const void* x, long long x_token_stride, long long x_head_stride, void* y,
                    long long y_token_stride, long long y_head_stride, int type, int t, int heads,
                    int head_dim, const int* pos, const strasgpt_rope_t* rope, void* stream) {
  return turn<RopeArgs>("strasgpt_k_rope", x, x_token_stride, x_head_stride, y, y_token_stride,
                        y_head_stride, type, t, heads, head_dim, pos, rope, stream,
                        [&](RopeArgs& a) -> const char* {
                          if (t == 0) return nullptr;
                          return turns_of(*rope, rope->dim / 2, a.turns, [](int m) { return m; })
                                     ? nullptr
                                     : kTooFast;
                        });
}

int strasgpt_k_rope_axes(const void* x, long long x_token_stride, long long x_head_stride, void* y,
                         long long y_token_stride, long long y_head_stride, int type, int t,
                         int heads, int head_dim, const int* pos, long long pos_axis_stride,
                         long long pos_token_stride, const strasgpt_rope_t* rope,
                         const strasgpt_rope_axes_t* axes, void* stream) {
  return turn<AxesArgs>(
      "strasgpt_k_rope_axes", x, x_token_stride, x_head_stride, y, y_token_stride, y_head_stride,
      type, t, heads, head_dim, pos, rope, stream, [&](AxesArgs& a) -> const char* {
        if (!axes) return "null axes";
        const int n = axes->axes, half = rope->dim / 2;
        if (n < 1 || n > STRASGPT_ROPE_AXES_MAX) return "1 to 4 axes";
        if (axes->order != STRASGPT_AXES_RUNS && axes->order != STRASGPT_AXES_DEALT)
          return "unknown order of the axes";
        long long sum = 0;
        for (int i = 0; i < n; i++) {
          if (axes->section[i] < 0) return "a section of fewer than 0 pairs";
          sum += axes->section[i];
        }
        if (sum != half) return "the sections must add up to the turned pairs";
        if (pos_axis_stride < 0 || pos_token_stride < 0) return "negative stride of pos";
        a.pa = pos_axis_stride;
        a.pt = pos_token_stride;
        // Pair of every axis's m-th.
        uint8_t pair[STRASGPT_ROPE_AXES_MAX][kMaxPairs];
        int given[STRASGPT_ROPE_AXES_MAX] = {};
        for (int j = 0, i = 0; j < half; j++) {
          while (given[i] == axes->section[i]) i = (i + 1) % n;
          a.axis[j] = (uint8_t)i;
          pair[i][given[i]++] = (uint8_t)j;
          if (axes->order == STRASGPT_AXES_DEALT) i = (i + 1) % n;
        }
        if (!axes->separate)
          return turns_of(*rope, half, a.turns, [](int m) { return m; }) ? nullptr : kTooFast;
        for (int i = 0; i < n; i++)
          if (axes->section[i] &&
              !turns_of(*rope, axes->section[i], a.turns, [&](int m) { return pair[i][m]; }))
            return kTooFast;
        return nullptr;
      });
}

}  // extern "C"
