// strasgpt_k_sample: one token per row of logits, from a given random number.
//
// Mathematics. With M the row's largest logit and T its temperature an entry
// weighs w = exp((x - M) / T). The filters keep a prefix of the order "larger
// logit first, equal ones by index": top-k its first k; top-p the shortest
// prefix of those that reaches p of their mass; min-p the entries with
// w >= min_p. The token is the first kept one, in index order, whose running
// mass exceeds u times the kept mass.
//
// Weights are 64-bit: 2^(n / 256) from a table times a cubic, 2^-42 relative.
// fp32 has an error of 1e-7 per weight, which moves a border between a
// hundred thousand tokens by more than many of them weigh. Sums that atomics
// gather are integers, in a unit of 2^-31 of the largest weight that can be
// in their bin of the histogram (two 16-bit halves of up to 45056 entries fit
// 32-bit sums), and all others are added in a fixed order: the same row gives
// the same bits whatever the order of CTAs and threads. A bin is less than 0.3
// octaves wide and its unit's power of two at most one octave above its largest
// weight, so a weight is rounded, to nearest, by at most 2^-30.7 of itself
// (below 2^-72 of the largest one: by 2^-104). Different weights' roundings
// mostly cancel; equal logits, as bf16 rows have by the thousand, round alike,
// and move a border by up to that much of the mass before it: 2e-4 of an entry
// in a flat row of 360448. Entries ranked next to a border have kFine bits more.
//
// A row is a thread-block cluster, each CTA holding a slice of it in shared
// memory: logits are read from HBM once, whatever the filters then need.
// First a bound drops what cannot be kept, so that 64-bit work is done for
// few entries:
//   top-k   an entry below the k-th largest of 1024 or fewer groups' largest
//           ones (the groups' maxima are exchanged with the row's own);
//   min-p   one below it.
// No sort of the row: one histogram over the logit's distance from M finds
// the bin in which a filter's border lies (a count for top-k, a mass for
// top-p); the entries of that bin, a few as a rule, are exchanged and ranked
// among themselves. A bin with more entries than kList is divided again, by
// distance and then by key, until few or only equal ones are left. Where
// top-k's bound leaves at most kThreads entries of the row, one CTA sorts
// those and does the rest. Many rows under top-k: see k_sample_rows.
//
// What bounds it, measured: one row of 128256 fp32 logits under top-k 50 takes
// 12 us, a chain of reading, two exchanges between CTAs, a sort. 64 rows of
// 151936 under top-p 0.95, 87 us: two rounds of CTAs, 31 us each, of which the
// histogram's 64-bit weights and shared-memory additions are 10 us (0.5 cycles
// an entry and SM), four exchanges 11, the division of the border's bin 4, the
// reading 3 (of the other 25 us a part is the launch in front, k_sample_rows;
// they were not taken apart further). 256 rows of 201088 bf16 logits under
// top-k 200, 53 us (1.9 TB/s; 16 us of bytes): two reads, the second from L2,
// and a sort per row. Slices read again from L2 instead of kept in shared
// memory were slower at every size (64 rows of 151936: 129 us).
#include <cooperative_groups.h>
#include <float.h>

#include "entry.h"

extern "C" {
#include "strasgpt_kernels.h"
}

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = kThreads;  // one per thread
constexpr int kGroups = kThreads / 4;  // of a CTA, whose maxima bound top-k
constexpr int kList = 256;       // entries ranked against each other
constexpr int kWords = 3;        // a thread's entries (at most 96) as bits
constexpr int kKept = 4096;      // entries of a slice listed behind a bound
constexpr int kUnit = 31;        // a weight in its bin's unit is at most 2^kUnit
constexpr int kFine = 11;        // bits more of the weights of ranked entries
constexpr int kReach = 72;       // octaves of weight that the bins divide evenly

struct SampleArgs {
  const void* logits;
  long long ld;
  int vocab, per;                // entries of a row, of a CTA's slice
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* token;
  float* prob;
  int* kept;
  int vec;                       // rows can be read 16 bytes at a time
  int pending;                   // only the rows that k_sample_rows left
};

struct Entry {
  unsigned key;
  int idx;
  u64 w;                         // in the bin's unit / 2^kFine
};

// What a CTA's threads share, before its slice of the row.
struct alignas(16) Shared {
  double table[256];             // 2^(i / 256)
  u64 gmass[kBins];              // histogram of the row: mass, count
  unsigned gcount[kBins];
  unsigned count[kBins];         // of this slice: count, and the mass as the
  unsigned lo[kBins], hi[kBins]; // sums of the weights' lower and upper 16 bits
  union {
    Entry list[2][kList];        // border entries of top-k, of top-p
    struct {
      u64 few[kThreads];         // the row's entries that the bound leaves,
      u64 order[kThreads];       // when they are few: key, index
    };
    struct {
      u64 gather_mass[kBins];    // a share of the bins from every CTA
      unsigned gather_count[kBins];
    };
  };
  union {
    float maxima[kMaxCluster * kGroups];  // the groups' largest logits
    unsigned short kept[kKept];  // places of the entries that a bound leaves
  };
  // One slot per CTA of the cluster, written by that CTA in all of them.
  float least[kMaxCluster];
  unsigned kmin[kMaxCluster], kmax[kMaxCluster];
  unsigned number[kMaxCluster];
  double mass[kMaxCluster];
  unsigned total[kMaxCluster];
  unsigned left[kMaxCluster];    // entries that the bound leaves in each slice
  u64 wred[kWarps];
  double wsum[kWarps];
  unsigned wmin[kWarps], wmax[kWarps];
  float wleast[kWarps];
  double before_mass[kMaxCluster];    // what each slice has before the border's
  unsigned before_count[kMaxCluster]; // entries, then what it keeps in all
  u64 slice_mass[kMaxCluster];   // of the border's entries, what is kept of
  unsigned slice_count[kMaxCluster];  // each slice
  unsigned few_count;
  double bbase;
  u64 bmass;
  unsigned bcount, bbin, fill;
  int found;
  unsigned cut_key;
  int cut_idx;
};

// Order-preserving key of a logit (never NaN here).
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ void store_f(float& to, float v) { to = v; }
__device__ __forceinline__ void store_f(uint16_t& to, float v) {
  to = (uint16_t)(__float_as_uint(v) >> 16);  // 0, or cut to bf16's lowest value
}
__device__ __forceinline__ float load_f(float v) { return v; }
__device__ __forceinline__ float load_f(uint16_t v) { return sg::bf16_to_f32(v); }

// A NaN or -inf logit is never taken; -0 equals 0, so it ranks as 0.
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }

__device__ __forceinline__ u64 shfl_up(u64 v, int o) { return __shfl_up_sync(0xFFFFFFFFu, v, o); }
__device__ __forceinline__ double shfl_up(double v, int o) {
  return __shfl_up_sync(0xFFFFFFFFu, v, o);
}

// Sums over the block in a fixed order; every thread gets its inclusive
// prefix and the total.
template <typename N>
__device__ __forceinline__ N block_prefix(N v, N* red, N* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N n = shfl_up(v, o);
    if (lane >= o) v += n;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  N w = lane < kWarps ? red[lane] : N(0);
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const N n = shfl_up(w, o);
    if (lane >= o) w += n;
  }
  *total = __shfl_sync(0xFFFFFFFFu, w, kWarps - 1);
  const N before = __shfl_sync(0xFFFFFFFFu, w, (warp + 31) & 31);
  return warp ? before + v : v;
}

// 2^e for -1022 <= e <= 1023.
__device__ __forceinline__ double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// Descending bitonic sort of the first n threads' values (the others' are 0
// and smaller than all); `x` holds kThreads words.
__device__ __forceinline__ u64 block_sort(u64 v, int n, u64* x) {
  const int i = threadIdx.x;
  for (int size = 2; size < 2 * n; size *= 2)
    for (int step = size / 2; step; step /= 2) {
      u64 o;
      if (step < 32) {
        o = __shfl_xor_sync(0xFFFFFFFFu, v, step);
      } else {
        __syncthreads();
        x[i] = v;
        __syncthreads();
        o = x[i ^ step];
      }
      const bool larger = ((i & size) == 0) == ((i & step) == 0);
      v = larger == (v > o) ? v : o;
    }
  return v;
}

// Where the running mass has to be exceeded. u at or above 1 takes the last
// entry with a weight, which roundings of the sums must not decide.
__device__ __forceinline__ double draw_at(float u, double total) {
  return u < 1.f ? (u > 0.f ? (double)u * total : 0.0) : u == u ? (double)INFINITY : 0.0;
}

// The choice of a row from its n <= kThreads entries that can be kept, one
// block's work. mark: this thread's entry, its key over INT_MAX - index (0
// behind the last). `few` and `order` hold kThreads words, `wsum` kWarps.
template <typename W>
__device__ __forceinline__ void finish(const SampleArgs& a, int row, u64 mark, int n, int k,
                                       float p, double min_w, float u, W weight, u64* few,
                                       u64* order, double* wsum, int* found, unsigned* fill) {
  // Sorted, entry `tid` of the order is thread tid's.
  const int tid = threadIdx.x;
  const bool real = tid < n;
  const u64 v = block_sort(mark, n, order);
  double w = real ? weight(of_key((unsigned)(v >> 32))) : 0.0;
  bool stays = real && tid < k;
  double mass;
  const double upto_w = block_prefix(stays ? w : 0.0, wsum, &mass);
  if (p < 1.f) stays = stays && (tid == 0 || upto_w - w < (double)p * mass);
  stays = stays && w >= min_w;
  const int kept = __syncthreads_count(stays);
  // What stays, by index.
  double* weights = reinterpret_cast<double*>(few);
  weights[tid] = w;
  const u64 byi = block_sort(stays ? (u64)(unsigned)v << 32 | (unsigned)tid : 0, n, order);
  __syncthreads();
  w = tid < kept ? weights[(unsigned)byi] : 0.0;
  double total;
  const double run = block_prefix(w, wsum, &total);
  const double target = draw_at(u, total);
  if (tid == 0) {
    *found = kThreads;
    *fill = 0;
  }
  __syncthreads();
  if (w > 0) {
    if (run > target) atomicMin(found, tid);
    atomicMax(fill, tid);
  }
  __syncthreads();
  if (tid == min(*found, (int)*fill)) {
    a.token[row] = INT_MAX - (int)(unsigned)(byi >> 32);
    if (a.prob) a.prob[row] = (float)(w / total);
    if (a.kept) a.kept[row] = kept;
  }
}

// Many rows under top-k: a block per row reads it twice, once for the largest
// logits of 1024 groups (two a thread), whose k-th largest bounds the row's,
// and once, in part from L2, for the entries above that bound, at most
// kThreads. No block waits for another. A row that this does not serve (no
// top-k up to kThreads, too many entries left, infinite logits) gets the token
// kPending and is the cluster kernel's.
constexpr int kPending = -2;

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample_rows(SampleArgs a) {
  __shared__ u64 few[kThreads], order[kThreads], wred[kWarps];
  __shared__ double wsum[kWarps];
  __shared__ float wtop[kWarps], wleast[kWarps];
  __shared__ unsigned count[kBins], fill, bin;
  __shared__ int found;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  sg::pdl_trigger();
  sg::pdl_wait();
  const float T_ = a.temperature ? a.temperature[row] : 1.f;
  const int k = a.top_k[row];
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const float min_p = a.min_p ? a.min_p[row] : 0.f;
  const bool greedy = !(T_ > 0.f) || k == 1 || p <= 0.f;
  if (k <= 0 || k > kThreads || k >= a.vocab) {
    if (tid == 0) a.token[row] = kPending;
    return;
  }
  const T* src = static_cast<const T*>(a.logits) + row * a.ld;
  constexpr int V = 16 / sizeof(T);
  const int nv = a.vec ? a.vocab / V : 0;
  // f(logit, index) for all of the row; a NaN or -inf fails its comparisons.
  // The second time from the end: what was read last is in L2 (256 rows of
  // 201088 bf16, 56.5 -> 53.4 us).
  auto each = [&](bool back, auto f) {
    const int number = nv > tid ? (nv - 1 - tid) / kThreads + 1 : 0;
    const int step = back ? -kThreads : kThreads;
    int v = back ? tid + (number - 1) * kThreads : tid;
#pragma unroll 4
    for (int left = number; left > 0; left--, v += step) {
      const uint4 r = reinterpret_cast<const uint4*>(src)[v];
      T e[V];
      memcpy(e, &r, 16);
#pragma unroll
      for (int j = 0; j < V; j++) f(load_f(e[j]), v * V + j);
    }
    for (int i = nv * V + tid; i < a.vocab; i += kThreads) f(load_f(src[i]), i);
  };
  float top[2] = {-INFINITY, -INFINITY};
  each(false, [&](float x, int i) { top[i & 1] = fmaxf(top[i & 1], x); });
  top[0] += 0.f;  // -0 is 0
  top[1] += 0.f;
  float M = fmaxf(top[0], top[1]);
  // The smallest of the groups' largest that are there.
  float least = fminf(top[0] > -INFINITY ? top[0] : INFINITY, top[1] > -INFINITY ? top[1] : INFINITY);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
    least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
  }
  if (lane == 0) {
    wtop[warp] = M;
    wleast[warp] = least;
  }
  count[tid] = 0;
  if (tid == 0) {
    fill = 0;
    bin = kBins;
    found = INT_MAX;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    M = fmaxf(M, wtop[w]);
    least = fminf(least, wleast[w]);
  }
  if (M == -INFINITY) {          // nothing but -inf and NaN
    if (tid == 0) {
      a.token[row] = -1;
      if (a.prob) a.prob[row] = 0.f;
      if (a.kept) a.kept[row] = 0;
    }
    return;
  }
  if (greedy) {
    // The largest, at its lowest index.
    int first = INT_MAX;
    each(true, [&](float x, int i) { first = x == M ? min(first, i) : first; });
    if (first < INT_MAX) atomicMin(&found, first);
    __syncthreads();
    if (tid == 0) {
      a.token[row] = found;
      if (a.prob) a.prob[row] = 1.f;
      if (a.kept) a.kept[row] = 1;
    }
    return;
  }
  if (M == INFINITY) {
    if (tid == 0) a.token[row] = kPending;
    return;
  }
  // The bin of the k-th largest group, and a logit just below that bin.
  const float bins_per = fminf((kBins - 1) / (M - least), 1e37f);
#pragma unroll
  for (int g = 0; g < 2; g++)
    if (top[g] > -INFINITY)
      atomicAdd(&count[(int)fminf((M - top[g]) * bins_per, (float)(kBins - 1))], 1u);
  __syncthreads();
  u64 all;
  const u64 upto = block_prefix((u64)count[tid], wred, &all);
  if (upto >= (u64)k) atomicMin(&bin, (unsigned)tid);
  __syncthreads();
  // Fewer groups than k: no bound but -inf's. The last bin ends at the
  // smallest group. (A range beyond fp32 has one bin and no bound either.)
  const float floor = fmaxf(
      -FLT_MAX, bin == kBins ? -FLT_MAX
                : bin == kBins - 1
                    ? least
                    : __double2float_rd((double)M - (bin + 1.01) / (double)bins_per -
                                        1e-6 * (fabs((double)M) + (double)(M - least))));
  each(true, [&](float x, int i) {
    if (x >= floor) {
      const unsigned at = atomicAdd(&fill, 1u);
      if (at < kThreads) few[at] = ((u64)key_of(x + 0.f) << 32) | (unsigned)(INT_MAX - i);
    }
  });
  __syncthreads();
  const unsigned n = fill;
  __syncthreads();               // before `fill` serves the choice
  if (n > kThreads) {
    if (tid == 0) a.token[row] = kPending;
    return;
  }
  const double scale = 1.4426950408889634 / (double)T_;
  const double min_w = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
  finish(a, row, tid < (int)n ? few[tid] : 0, (int)n, k, p, min_w, a.u[row],
         [&](float x) { return exp2(((double)x - (double)M) * scale); }, few, order, wsum, &found,
         &fill);
}

template <typename T>
struct Row {
  Shared* sh;
  const T* xs;                   // this CTA's slice
  int n;                         // its entries
  cg::cluster_group cluster;
  int rank, ranks;
  int start, per;                // the slice's first index, a slice's length
  int c0, c1;                    // this thread's entries [c0, c1) of it, or
  bool listed;                   // of those listed in sh->kept
  float floor;                   // entries below are out
  float M;
  double scale;                  // log2(e) / T
  bool ends;                     // u near 0, or not below 1: the smallest weight counts
  float shrink;                  // distances are measured times this
  float bins_per;                // histogram bins per unit of that
  float octaves;                 // octaves of weight per bin
  float last;                    // bins from M to where a bin's unit is far above the weights
  float gone;                    // logits up to here weigh less than e^-749, 0 in 64 bits

  __device__ float at(int i) const { return clean(load_f(xs[i])); }

  // f(four logits, place of the first) for all of the slice, in any order;
  // behind the last, -inf.
  template <typename F>
  __device__ __forceinline__ void fours(F f) const {
    constexpr int V = 16 / sizeof(T);
    for (int v = threadIdx.x; v * V < n; v += kThreads) {
      const uint4 r = reinterpret_cast<const uint4*>(xs)[v];
      T e[V];
      memcpy(e, &r, 16);
#pragma unroll
      for (int h = 0; h < V; h += 4) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = v * V + h + j < n ? load_f(e[h + j]) : -INFINITY;
        f(x, v * V + h);
      }
    }
  }

  // Drops the entries below `least` (and -inf) and returns how many stay. Up
  // to kKept of them are listed, so that the threads get equal shares;
  // otherwise each thread keeps its part of the slice.
  __device__ unsigned bound(float least) {
    floor = fmaxf(least, -FLT_MAX);
    unsigned in[kWords], mine = 0;
#pragma unroll
    for (int w = 0; w < kWords; w++) {
      unsigned m = 0;
      const int a = c0 + 32 * w, n = min(32, c1 - a);
#pragma unroll 8
      for (int j = 0; j < n; j++) m |= (unsigned)(load_f(xs[a + j]) >= floor) << j;
      in[w] = m;
      mine += __popc(m);
    }
    u64 total;
    unsigned at = (unsigned)block_prefix((u64)mine, sh->wred, &total) - mine;
    listed = total <= kKept;
    if (listed) {
#pragma unroll
      for (int w = 0; w < kWords; w++)
        for (unsigned m = in[w]; m; m &= m - 1)
          sh->kept[at++] = (unsigned short)(c0 + 32 * w + __ffs(m) - 1);
      const int share = ((int)total + kThreads - 1) / kThreads;
      c0 = min((int)threadIdx.x * share, (int)total);
      c1 = min(c0 + share, (int)total);
      __syncthreads();
    }
    return (unsigned)total;
  }
  __device__ int place(int j) const { return listed ? sh->kept[j] : j; }
  // f(logit, place in the slice) for what is left, in index order.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int j = c0; j < c1; j++) {
      const int i = place(j);
      const float x = at(i);
      if (x >= floor) f(x, i);
    }
  }

  // Distance from M in bins (-inf and NaN: FLT_MAX). Every step is monotone,
  // so larger logits come first whatever the roundings.
  __device__ float distance(float x) const { return fmaf(x, -shrink, M * shrink); }
  __device__ float pos(float x) const { return fminf(distance(x) * bins_per, FLT_MAX); }
  // The integer below, by adding 2^23 rounded down.
  __device__ static int whole(float f) { return __float_as_int(__fadd_rd(f, 8388608.f)) & 0x7FFFFF; }
  // Histogram bin; the last one is open to below.
  __device__ static int bin_at(float f) { return whole(fminf(f, (float)(kBins - 1))); }
  __device__ int bin_of(float x) const { return bin_at(pos(x)); }
  // The weights of bin b are at most 2^-e: their unit is 2^-(e + kUnit).
  __device__ int unit_of(int b) const { return kUnit + whole((float)b * octaves); }

  // exp((x - M) / T) as v p 2^e, with 1 <= v < 2 and p nearly 1. 2^t with t in
  // units of 1/256 taken apart by adding 1.5 * 2^44, a cubic for the rest
  // (|r ln 2| < 1.4e-3, the next term is below 1.5e-13). No branches, so that a
  // loop's weights overlap.
  __device__ double power(float x, double* p, int* e) const {
    const double d = (double)x - (double)M;
    const double magic = 6755399441055744.0 / 256;
    const double z = fma(d, scale, magic);
    const int n = __double2loint(z);
    const double r = fma(d, scale, magic - z);
    *p = fma(fma(fma(r, 0.05550410866482158, 0.2402265069591007), r, 0.6931471805599453), r, 1.0);
    *e = n >> 8;
    return sh->table[n & 255];
  }
  __device__ static double shifted(double v, int e) {
    return __hiloint2double(__double2hiint(v) + e * (1 << 20), __double2loint(v));
  }
  // The weight; 0 where 64 bits round it to 0 (and for -inf and NaN). The last
  // factor makes the subnormal ones.
  __device__ double weight(float x) const {
    int e;
    double p;
    const double v = power(x, &p, &e);
    return x > gone ? shifted(v * p, e + 128) * 0x1p-128 : 0.0;
  }
  // A weight in units of 2^-unit, rounded: adding 2^52 leaves the nearest
  // integer in the low 52 bits. (A rounding of the bin's border may let a
  // weight exceed 2^kUnit by a little.)
  __device__ u64 in_units(double w, int unit) const {
    return (u64)__double_as_longlong(fma(w, pow2(unit), 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }
  // The weight of x, f bins from M, in a bin's unit (0 far below the bins'
  // units).
  __device__ unsigned units(float x, float f, int unit) const {
    int e;
    double p;
    const double v = power(x, &p, &e);
    const unsigned w = (unsigned)__double2loint(fma(shifted(v, e + unit), p, 4503599627370496.0));
    return f < last ? w : 0u;
  }
  __device__ void add(int b, unsigned w) {
    if (w == 0) return;
    atomicAdd(&sh->lo[b], w & 0xFFFFu);
    atomicAdd(&sh->hi[b], w >> 16);
  }
  __device__ static u64 join(unsigned lo, unsigned hi) { return ((u64)hi << 16) + lo; }
  __device__ void clear() {
    sh->count[threadIdx.x] = sh->lo[threadIdx.x] = sh->hi[threadIdx.x] = 0;
    __syncthreads();
  }

  // The histogram of what is left, with counts.
  __device__ void histogram() {
    clear();
    each([&](float x, int) {
      const float f = pos(x);
      const int b = bin_at(f);
      atomicAdd(&sh->count[b], 1u);
      add(b, units(x, f, unit_of(b)));
    });
    gather_histogram();
  }
  // The masses alone, of all of the row.
  __device__ void histogram_of_all() {
    clear();
    // Four entries' weights side by side, then their additions.
    fours([&](const float* x, int) {
      unsigned w[4];
      int b[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float f = pos(x[j]);
        // bin_at and unit_of, without a conversion.
        const float z = __fadd_rd(fminf(f, (float)(kBins - 1)), 8388608.f);
        b[j] = __float_as_int(z) & 0x7FFFFF;
        w[j] = units(x[j], f, kUnit + whole((z - 8388608.f) * octaves));
      }
#pragma unroll
      for (int j = 0; j < 4; j++) add(b[j], w[j]);
    });
    gather_histogram();
  }
  // The slices' histograms become the row's, in every CTA: each adds up its
  // share of the bins and hands it to all. A warp reads, and writes, one other
  // CTA's neighbouring bins.
  __device__ void gather_histogram() {
    cluster.sync();
    const int share = kBins / ranks, at = threadIdx.x & (share - 1), b = rank * share + at;
    Shared* o = cluster.map_shared_rank(sh, threadIdx.x / share);
    unsigned c = o->count[b];
    u64 m = join(o->lo[b], o->hi[b]);
    if (ranks > 1) {
      sh->gather_count[threadIdx.x] = c;
      sh->gather_mass[threadIdx.x] = m;
      __syncthreads();
      c = 0;
      m = 0;
      for (int r = 0; r < ranks; r++) {
        c += sh->gather_count[r * share + at];
        m += sh->gather_mass[r * share + at];
      }
    }
    o->gcount[b] = c;
    o->gmass[b] = m;
    cluster.sync();
  }

  // The mass of a bin of the whole row's histogram.
  __device__ double mass_of(int b) const { return (double)sh->gmass[b] * pow2(-unit_of(b)); }

  // The row's mass, from its histogram.
  __device__ double mass() {
    double all;
    block_prefix(mass_of(threadIdx.x), sh->wsum, &all);
    return all;
  }

  // The lowest bin whose thread says so; kBins: none.
  __device__ unsigned first_bin(bool here) {
    if (threadIdx.x == 0) sh->bbin = kBins;
    __syncthreads();
    const unsigned who = __ballot_sync(0xFFFFFFFFu, here);
    if (who && (threadIdx.x & 31) == __ffs(who) - 1) atomicMin(&sh->bbin, threadIdx.x);
    __syncthreads();
    return sh->bbin;
  }

  // The bin with the border: the first whose entries bring the count to k
  // (by_mass: the mass to target; a bin without mass is no border, whatever
  // its sums' roundings say). Leaves it in sh->bbin, the count before it in
  // sh->bcount, the mass in sh->bbase; false: no bin does.
  __device__ bool find_bin(bool by_mass, double target, unsigned k) {
    const unsigned c = sh->gcount[threadIdx.x];
    const double m = mass_of(threadIdx.x);
    u64 all;
    double mall;
    const unsigned upto = (unsigned)block_prefix((u64)c, sh->wred, &all);
    const double mupto = block_prefix(m, sh->wsum, &mall);
    const unsigned bin = first_bin(by_mass ? m > 0 && mupto >= target : c && upto >= k);
    if (bin == threadIdx.x) {
      sh->bcount = upto - c;
      sh->bbase = mupto - m;
    }
    __syncthreads();
    return bin < kBins;
  }

  // The same within one bin of the row's histogram: integers, on top of
  // `count`, `base` and `mass` before it; the mass goes to sh->bmass.
  __device__ void find_sub_bin(bool by_mass, double target, unsigned k, unsigned count,
                               double base, u64 mass, double unit) {
    const unsigned c = sh->gcount[threadIdx.x];
    const u64 m = sh->gmass[threadIdx.x];
    u64 all;
    const unsigned upto = count + (unsigned)block_prefix((u64)c, sh->wred, &all);
    const u64 mupto = mass + block_prefix(m, sh->wred, &all);
    unsigned bin = first_bin(c && (by_mass ? base + (double)mupto * unit >= target : upto >= k));
    if (bin == kBins) {
      // Roundings of the row's sums left the border behind the bin's last
      // entry: that one it is.
      __syncthreads();
      if (threadIdx.x == 0) sh->bbin = 0;
      __syncthreads();
      if (c) atomicMax(&sh->bbin, threadIdx.x);
      __syncthreads();
      bin = sh->bbin;
    }
    if (bin == threadIdx.x) {
      sh->bcount = upto - c;
      sh->bmass = mupto - m;
    }
    __syncthreads();
  }

  // First index of this slice, in index order, at which the running sum of
  // `value(x, i)` exceeds `target`; the last with a value if roundings leave
  // none. upto: the inclusive prefix of this thread's sum `mine`, of which
  // one in the block is positive.
  template <typename F>
  __device__ int find_index(F value, double mine, double upto, double target) {
    if (threadIdx.x == 0) {
      sh->found = 2 * kThreads;
      sh->fill = 0;
    }
    __syncthreads();
    if (mine > 0) {
      if (upto > target) atomicMin(&sh->found, (int)threadIdx.x);
      atomicMax(&sh->fill, threadIdx.x);
    }
    __syncthreads();
    const int owner = min(sh->found, (int)sh->fill);
    __syncthreads();
    // The owner's warp looks at its entries together.
    if (owner >> 5 == threadIdx.x >> 5) {
      const int lane = threadIdx.x & 31, from = owner & 31;
      double run = __shfl_sync(0xFFFFFFFFu, upto - mine, from);
      const int a = __shfl_sync(0xFFFFFFFFu, c0, from), b = __shfl_sync(0xFFFFFFFFu, c1, from);
      int last = -1;
      for (int j0 = a; j0 < b; j0 += 32) {
        const int i = place(min(j0 + lane, b - 1));
        const double v = j0 + lane < b ? value(at(i), start + i) : 0.0;
        double s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double n = shfl_up(s, o);
          if (lane >= o) s += n;
        }
        const unsigned some = __ballot_sync(0xFFFFFFFFu, v > 0);
        const unsigned over = __ballot_sync(0xFFFFFFFFu, v > 0 && run + s > target);
        if (some) last = j0 + 31 - __clz(some);
        if (over) {
          last = j0 + __ffs(over) - 1;
          break;
        }
        run += __shfl_sync(0xFFFFFFFFu, s, 31);
      }
      if (lane == 0) sh->found = place(last);
    }
    __syncthreads();
    return start + sh->found;
  }

  // The prefix of the order that a filter keeps: its last entry (key and
  // index) and its mass. tail: the border lies among entries whose weight the
  // histogram rounds to 0; all others are kept, and `zeros` of those. sums:
  // sh->before_mass and sh->before_count say what is kept of each slice.
  struct Cut {
    unsigned key;
    int idx;
    double mass;
    bool tail, sums;
    unsigned zeros;
  };

  // by_mass: the shortest prefix whose mass reaches `target`; else the first
  // k. The row's histogram is there.
  __device__ Cut select(bool by_mass, double target, unsigned k, bool& ready, int which) {
    Cut cut = {0u, INT_MAX, 0.0, false, false, 0u};
    if (!find_bin(by_mass, target, k)) {  // fewer than k entries: all are kept
      cut.mass = mass();
      return cut;
    }
    const int bin = (int)sh->bbin, unit = unit_of(bin);
    const double step = pow2(-unit), base = sh->bbase;
    unsigned count = sh->bcount, number = sh->gcount[bin];
    u64 mass = 0;                         // within the bin, before its border
    if (!by_mass && bin == kBins - 1 && sh->gmass[bin] == 0 && !ends) {
      cut.tail = true;
      cut.zeros = k - count;
      cut.mass = base;
      return cut;
    }
    // The entries in question: a range of distances, and of keys.
    float from = (float)bin, to = bin < kBins - 1 ? (float)(bin + 1) : INFINITY;
    unsigned lo = 0, hi = 0xFFFFFFFFu;
    int digit = bin;
    bool few = false;                     // sh->kept lists them
    unsigned own = 0;                     // how many are this slice's
    auto in_set = [&](float x) {
      const float f = pos(x);
      if (!(f >= from && f < to)) return false;
      const unsigned key = key_of(x);
      return key >= lo && key <= hi;
    };
    if (by_mass || number > kList) {
      // Divide the bin evenly (f - bin and its multiple are exact). On the
      // way: what the slice has before it.
      double slice, fine;
      block_prefix((int)threadIdx.x < bin ? (double)join(sh->lo[threadIdx.x], sh->hi[threadIdx.x]) *
                                                pow2(-unit_of(threadIdx.x))
                                          : 0.0,
                   sh->wsum, &slice);
      unsigned above = 0;
      if (threadIdx.x == 0) sh->fill = 0;
      clear();
      auto divide = [&](float x, float f) {
        const int d = bin_at((f - from) * kBins);
        atomicAdd(&sh->count[d], 1u);
        add(d, units(x, f, unit));
      };
      if (listed) {
        each([&](float x, int) {
          const float f = pos(x);
          above += f < from;
          if (f >= from && f < to) divide(x, f);
        });
      } else {
        // The bin's entries are listed for the last look at them.
        fours([&](const float* x, int i) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float f = pos(x[j]);
            above += f < from;
            if (f >= from && f < to && x[j] >= floor) {
              divide(x[j], f);
              const unsigned p = atomicAdd(&sh->fill, 1u);
              if (p < kKept) sh->kept[p] = (unsigned short)(i + j);
            }
          }
        });
      }
      gather_histogram();
      own = sh->fill;
      few = !listed && own <= kKept;
      ready = false;
      find_sub_bin(by_mass, target, k, count, base, mass, step);
      digit = (int)sh->bbin;
      count = sh->bcount;
      mass = sh->bmass;
      number = sh->gcount[digit];
      const bool before = (int)threadIdx.x < digit;
      block_prefix(before ? (double)join(sh->lo[threadIdx.x], sh->hi[threadIdx.x]) : 0.0, sh->wsum,
                   &fine);
      u64 counts;
      block_prefix((u64)(above + (before ? sh->count[threadIdx.x] : 0u)), sh->wred, &counts);
      if (threadIdx.x < ranks) {
        Shared* o = cluster.map_shared_rank(sh, threadIdx.x);
        o->before_mass[rank] = slice + fine * step;
        o->before_count[rank] = (unsigned)counts;
      }
      if (digit < kBins - 1) to = from + (float)(digit + 1) / kBins;
      from += (float)digit / kBins;
      cut.sums = true;
    }
    while (number > kList) {
      cut.sums = false;
      unsigned kmin = 0xFFFFFFFFu, kmax = 0, mine = 0;
      each([&](float x, int) {
        if (!in_set(x)) return;
        mine++;
        const unsigned key = key_of(x);
        kmin = min(kmin, key);
        kmax = max(kmax, key);
      });
      kmin = __reduce_min_sync(0xFFFFFFFFu, kmin);
      kmax = __reduce_max_sync(0xFFFFFFFFu, kmax);
      if ((threadIdx.x & 31) == 0) {
        sh->wmin[threadIdx.x >> 5] = kmin;
        sh->wmax[threadIdx.x >> 5] = kmax;
      }
      double total;
      const double upto = block_prefix((double)mine, sh->wsum, &total);
      if (threadIdx.x < ranks) {
        for (int w = 0; w < kWarps; w++) {
          kmin = min(kmin, sh->wmin[w]);
          kmax = max(kmax, sh->wmax[w]);
        }
        Shared* o = cluster.map_shared_rank(sh, threadIdx.x);
        o->kmin[rank] = kmin;
        o->kmax[rank] = kmax;
        o->number[rank] = (unsigned)total;
      }
      cluster.sync();
      kmin = 0xFFFFFFFFu;
      kmax = 0;
      unsigned before = 0;
      for (int r = 0; r < ranks; r++) {
        kmin = min(kmin, sh->kmin[r]);
        kmax = max(kmax, sh->kmax[r]);
        if (r < rank) before += sh->number[r];
      }
      if (kmin == kmax) {
        // Equal logits only: the first `take` by index are kept, while the
        // mass before them is below the target.
        const double w = weight(of_key(kmin)), ahead = base + (double)mass * step;
        unsigned take = by_mass ? number : k - count;
        if (by_mass && w > 0) {
          const double need = (target - ahead) / w;
          if (need < (double)number) take = need > 1.0 ? (unsigned)ceil(need) : 1u;
        }
        cut.key = kmin;
        cut.mass = ahead + take * w;
        if (take < number) {
          // The take-th of them lies in one slice.
          if (before < take && take <= before + (unsigned)total) {
            const int i = find_index(
                [&](float x, int) { return x >= floor && in_set(x) ? 1.0 : 0.0; }, (double)mine,
                upto, (double)(take - 1 - before));
            if (threadIdx.x < ranks) cluster.map_shared_rank(sh, threadIdx.x)->cut_idx = i;
          }
          cluster.sync();
          cut.idx = sh->cut_idx;
        }
        return cut;
      }
      int shift = 0;
      while (((kmax - kmin) >> shift) >= (unsigned)kBins) shift++;
      clear();
      each([&](float x, int) {
        if (!in_set(x)) return;
        const int d = (int)((kmax - key_of(x)) >> shift);
        atomicAdd(&sh->count[d], 1u);
        add(d, units(x, pos(x), unit));
      });
      gather_histogram();
      find_sub_bin(by_mass, target, k, count, base, mass, step);
      digit = (int)sh->bbin;
      count = sh->bcount;
      mass = sh->bmass;
      number = sh->gcount[digit];
      const u64 low = ((u64)(digit + 1) << shift) - 1, span = kmax - kmin;
      hi = kmax - ((unsigned)digit << shift);
      lo = kmax - (unsigned)(low < span ? low : span);
    }
    // The set's entries go to every CTA, this CTA's behind those of the CTAs
    // before it, and are ranked there.
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned before = 0;
      for (int r = 0; r < rank; r++) before += cluster.map_shared_rank(sh, r)->count[digit];
      sh->fill = before;
    }
    if (threadIdx.x < ranks) {
      sh->slice_mass[threadIdx.x] = 0;
      sh->slice_count[threadIdx.x] = 0;
    }
    __syncthreads();
    auto send = [&](float x, int i) {
      if (!in_set(x)) return;
      const unsigned p = atomicAdd(&sh->fill, 1u);
      const Entry e = {key_of(x), start + i, in_units(weight(x), unit + kFine)};
      for (int r = 0; r < ranks; r++) cluster.map_shared_rank(sh, r)->list[which][p] = e;
    };
    if (few) {
      for (unsigned j = threadIdx.x; j < own; j += kThreads) send(at(sh->kept[j]), sh->kept[j]);
    } else {
      each(send);
    }
    cluster.sync();
    const double ahead = base + (double)mass * step, fine = pow2(-unit - kFine);
    bool kept = false;
    unsigned place = 0;
    u64 before = 0;
    Entry e = {0u, 0, 0ull};
    if (threadIdx.x < number) {
      e = sh->list[which][threadIdx.x];
      for (unsigned j = 0; j < number; j++) {
        const Entry o = sh->list[which][j];
        if (o.key > e.key || (o.key == e.key && o.idx < e.idx)) {
          place++;
          before += o.w;
        }
      }
      // The border is in this set: its first entry is kept.
      kept = place == 0 ||
             (by_mass ? ahead + (double)before * fine < target : count + place < k);
      if (kept) {
        atomicAdd(&sh->slice_mass[e.idx / per], e.w);
        atomicAdd(&sh->slice_count[e.idx / per], 1u);
      }
    }
    const unsigned keeps = __syncthreads_count(kept);
    if (kept && place == keeps - 1) {
      sh->cut_key = e.key;
      sh->cut_idx = e.idx;
      sh->bmass = before + e.w;
    }
    if (cut.sums && threadIdx.x < ranks) {
      sh->before_mass[threadIdx.x] += (double)sh->slice_mass[threadIdx.x] * fine;
      sh->before_count[threadIdx.x] += sh->slice_count[threadIdx.x];
    }
    __syncthreads();
    cut.key = sh->cut_key;
    cut.idx = sh->cut_idx;
    cut.mass = ahead + (double)sh->bmass * fine;
    return cut;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared* sh = reinterpret_cast<Shared*>(raw);
  T* xs = reinterpret_cast<T*>(raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (a.pending) {
    sg::pdl_trigger();
    sg::pdl_wait();
    if (a.token[row] != kPending) return;
  }
  cluster.barrier_arrive();  // waited for before the first access to another CTA
  if (threadIdx.x < 256) sh->table[threadIdx.x] = exp2(threadIdx.x / 256.0);
  sg::pdl_trigger();
  sg::pdl_wait();

  const int start = min(rank * a.per, a.vocab), n = min(a.per, a.vocab - start);
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + start;
  // Slice into shared memory; its largest logit and its smallest finite one.
  float top = -INFINITY, least = INFINITY;
  auto take = [&](float x) {
    top = fmaxf(top, x);         // a NaN is passed over
    least = fminf(least, x > -INFINITY ? x : INFINITY);
  };
  constexpr int V = 16 / sizeof(T);
  const int nv = a.vec ? n / V : 0;
#pragma unroll 8
  for (int v = threadIdx.x; v < nv; v += kThreads) {
    const uint4 r = sg::ldg_stream(src + v * V);
    T e[V];
    memcpy(e, &r, 16);
#pragma unroll
    for (int j = 0; j < V; j++) take(load_f(e[j]));
    reinterpret_cast<uint4*>(xs)[v] = r;
  }
  for (int i = nv * V + threadIdx.x; i < n; i += kThreads) {
    xs[i] = src[i];
    take(load_f(xs[i]));
  }
  // The largest of each group of four threads goes to every CTA.
  top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
#pragma unroll
  for (int o = 16; o; o >>= 1) least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
  if (lane == 0) sh->wleast[warp] = least;
  if (threadIdx.x == 0) sh->few_count = 0;
  __syncthreads();
  cluster.barrier_wait();
  for (int q = lane & 3; q < ranks; q += 4)
    cluster.map_shared_rank(sh, q)->maxima[rank * kGroups + (threadIdx.x >> 2)] = top;
  if (threadIdx.x < ranks) {
#pragma unroll
    for (int w = 0; w < kWarps; w++) least = fminf(least, sh->wleast[w]);
    cluster.map_shared_rank(sh, threadIdx.x)->least[rank] = least;
  }
  float T_ = a.temperature ? a.temperature[row] : 1.f;
  const int k_ = a.top_k ? a.top_k[row] : 0;
  const float p_ = a.top_p ? a.top_p[row] : 1.f;
  const float m_ = a.min_p ? a.min_p[row] : 0.f;
  const float u_ = a.u[row];
  cluster.sync();
  least = INFINITY;
  for (int r = 0; r < ranks; r++) least = fminf(least, sh->least[r]);
  // Each warp looks at all groups: the row's largest logit, and the first
  // slice that has it.
  top = -INFINITY;
  for (int g = lane; g < ranks * kGroups; g += 32) top = fmaxf(top, sh->maxima[g]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  top += 0.f;                    // -0 is 0
  if (top == -INFINITY) {        // nothing but -inf and NaN
    if (rank == 0 && threadIdx.x == 0) {
      a.token[row] = -1;
      if (a.prob) a.prob[row] = 0.f;
      if (a.kept) a.kept[row] = 0;
    }
    return;
  }
  if (!(T_ > 0.f) || k_ == 1 || p_ <= 0.f) {
    // The largest, at its lowest index.
    int first = ranks;
    for (int g = lane; g < ranks * kGroups; g += 32)
      if (sh->maxima[g] == top) first = min(first, g / kGroups);
    if (rank != __reduce_min_sync(0xFFFFFFFFu, first)) return;
    if (threadIdx.x == 0) sh->found = INT_MAX;
    __syncthreads();
    int i = threadIdx.x;
    while (i < n && load_f(xs[i]) != top) i += kThreads;
    if (i < n) atomicMin(&sh->found, i);
    __syncthreads();
    if (threadIdx.x == 0) {
      a.token[row] = start + sh->found;
      if (a.prob) a.prob[row] = 1.f;
      if (a.kept) a.kept[row] = 1;
    }
    return;
  }

  const int chunk = ((a.per + kThreads - 1) / kThreads) | 1;  // odd: no bank conflicts
  Row<T> r{sh, xs, n, cluster, rank, ranks, start, a.per};
  r.c0 = min((int)threadIdx.x * chunk, n);
  r.c1 = min(r.c0 + chunk, n);
  if (top == INFINITY) {
    // Infinite logits share all of the mass: they become 0, the others the
    // lowest value, at a temperature of 1.
    T_ = 1.f;
    for (int i = r.c0; i < r.c1; i++) {
      const float x = load_f(xs[i]);
      if (x > -INFINITY) store_f(xs[i], x == INFINITY ? 0.f : -FLT_MAX);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < ranks * kGroups; g += kThreads)
      if (sh->maxima[g] > -INFINITY) sh->maxima[g] = sh->maxima[g] == INFINITY ? 0.f : -FLT_MAX;
    __syncthreads();
    top = 0.f;
    least = -FLT_MAX;
  }
  r.M = top;
  r.listed = false;
  // What the histogram rounds to 0, below 2^-104 of the largest weight, comes
  // to less than 2^-85 in all: only a u outside [2^-50, 1) can draw it.
  r.ends = !(u_ >= 0x1p-50f && u_ < 1.f);
  r.floor = -FLT_MAX;
  r.scale = 1.4426950408889634 / (double)T_;
  // The bins share what is within kReach octaves of the largest weight, or
  // down to the smallest logit if that is nearer. (Bins in 32 bits: all CTAs
  // compute the same ones, and any monotone ones do.)
  // Distances that fp32 might not hold are measured as quarters: then no step
  // below overflows, whatever the temperature. (M - x is one rounding either
  // way; a quarter is exact but for a denormal M, whose distance rounds to 0.)
  r.shrink = r.M - least <= FLT_MAX / 4 ? 1.f : 0.25f;
  const float bits = (float)fmin(r.scale / r.shrink, 1e37);
  const float range = fminf(kReach / bits, r.distance(least) * 1.00001f);
  r.bins_per = fminf((kBins - 1) / range, 1e37f);
  r.octaves = fminf(bits / r.bins_per, 2.0f * kReach / kBins);
  r.last = fminf(1000.f / (bits / r.bins_per), 1e38f);
  r.gone = fminf(__double2float_rd((double)r.M - 749.0 * (double)T_), of_key(key_of(r.M) - 1));
  const double min_w = m_ > 0.f ? fmin((double)m_, 1.0) : 0.0;
  // A logit just below M + T ln(w).
  auto logit_of = [&](double w) {
    return __double2float_rd((double)r.M + log2(w) * (1 + 1e-12) / r.scale - 1e-12 * fabs(r.M));
  };

  typename Row<T>::Cut cut = {0u, INT_MAX, 0.0, false, false, 0u};
  bool ready = false;
  if (k_ > 1 && k_ < a.vocab) {
    // The k-th largest of the groups' largest logits is not above the k-th
    // largest of all: find its bin.
    sh->gcount[threadIdx.x] = 0;
    sh->gmass[threadIdx.x] = 0;
    __syncthreads();
    for (int g = threadIdx.x; g < ranks * kGroups; g += kThreads) {
      const float x = sh->maxima[g] + 0.f;
      if (x > -INFINITY) atomicAdd(&sh->gcount[r.bin_of(x)], 1u);
    }
    __syncthreads();
    float least_kept = -INFINITY;
    if (k_ <= ranks * kGroups && r.find_bin(false, 0.0, (unsigned)k_)) {
      // Everything down to that bin's end stays.
      const int b = (int)sh->bbin;
      if (b < kBins - 1)
        least_kept = __double2float_rd((double)r.M -
                                       (b + 1.01) / ((double)r.bins_per * r.shrink) -
                                       1e-6 * (fabs((double)r.M) + (double)range / r.shrink));
    }
    const unsigned mine = r.bound(least_kept);
    // How many of the row are left; this slice's go to CTA 0 if it has few.
    Shared* o = cluster.map_shared_rank(sh, 0);
    if (threadIdx.x < ranks) cluster.map_shared_rank(sh, threadIdx.x)->left[rank] = mine;
    if (mine <= kThreads) {
      if (threadIdx.x == 0) sh->fill = atomicAdd(&o->few_count, mine);
      __syncthreads();
      r.each([&](float x, int i) {
        const unsigned at = atomicAdd(&sh->fill, 1u);
        if (at < kThreads) o->few[at] = ((u64)key_of(x) << 32) | (unsigned)(INT_MAX - start - i);
      });
    }
    cluster.sync();
    unsigned all = 0;
    for (int q = 0; q < ranks; q++) all += sh->left[q];
    if (all <= kThreads) {
      // Few: CTA 0 does the rest alone. Sorted, entry `tid` of the order is
      // thread tid's.
      if (rank > 0) return;
      const int tid = threadIdx.x;
      finish(a, row, tid < (int)all ? sh->few[tid] : 0, (int)all, k_, p_, min_w, u_,
             [&](float x) { return r.weight(x); }, sh->few, sh->order, sh->wsum, &sh->found,
             &sh->fill);
      return;
    }
    r.histogram();
    ready = true;
    cut = r.select(false, 0.0, (unsigned)k_, ready, 0);
    if (p_ < 1.f) {
      if (!ready) r.histogram();
      cut = r.select(true, (double)p_ * cut.mass, 0u, ready, 1);
    }
  } else if (p_ < 1.f) {
    r.histogram_of_all();
    cut = r.select(true, (double)p_ * r.mass(), 0u, ready, 1);
  } else {
    r.bound(min_w > 0 ? logit_of(min_w * 0.999) : -INFINITY);
  }
  // min-p counts where it drops the last entry that is kept so far.
  if (min_w > 0 && cut.sums) cut.sums = r.weight(of_key(cut.key)) >= min_w;

  // What is kept, in index order.
  auto kept_weight = [&](float x, int i, bool& kept) -> double {
    kept = false;
    if (!(x > -INFINITY)) return 0.0;
    if (cut.tail) {
      if (r.bin_of(x) == kBins - 1) return 0.0;
    } else {
      const unsigned key = key_of(x);
      if (key < cut.key || (key == cut.key && i > cut.idx)) return 0.0;
    }
    const double w = r.weight(x);
    kept = w >= min_w;
    return kept ? w : 0.0;
  };
  double mine = 0, upto = 0;
  auto add_up = [&](u64* numbers) {
    int number = 0;
    r.each([&](float x, int i) {
      bool kept;
      mine += kept_weight(x, start + i, kept);
      number += kept;
    });
    double total;
    upto = block_prefix(mine, sh->wsum, &total);
    if (numbers) block_prefix((u64)number, sh->wred, numbers);
    return total;
  };
  const bool known = cut.sums && !r.ends;  // what each slice keeps
  if (!known) {
    u64 numbers;
    const double total = add_up(&numbers);
    if (threadIdx.x < ranks) {
      Shared* o = cluster.map_shared_rank(sh, threadIdx.x);
      o->mass[rank] = total;
      o->total[rank] = (unsigned)numbers;
    }
    cluster.sync();
  }
  const double* slices = known ? sh->before_mass : sh->mass;
  double total = 0;
  unsigned kept = 0;
  for (int q = 0; q < ranks; q++) {
    total += slices[q];
    kept += known ? sh->before_count[q] : sh->total[q];
  }
  // The slice in which the running mass exceeds u total; the last with any
  // if none (u at or above 1).
  const double target = draw_at(u_, total);
  double run = 0, before = 0;
  int owner = -1;
  for (int q = 0; q < ranks; q++) {
    const double v = slices[q];
    if (v > 0 && (owner < 0 || !(run > target))) {
      owner = q;
      before = run;
    }
    run += v;
  }
  if (rank != owner) return;
  if (known) add_up(nullptr);
  const int token = r.find_index(
      [&](float x, int i) {
        bool in;
        return kept_weight(x, i, in);
      },
      mine, upto, target - before);
  if (threadIdx.x == 0) {
    a.token[row] = token;
    if (a.prob) a.prob[row] = (float)(r.weight(r.at(token - start)) / total);
    if (a.kept) a.kept[row] = (int)(kept + (cut.tail && min_w == 0 ? cut.zeros : 0u));
  }
}

// A slice that leaves room for two CTAs on an SM.
constexpr int kSliceBytes = 78 * 1024;

template <typename T>
cudaError_t launch(SampleArgs a, int rows, int cluster, int sms, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  const size_t smem = sizeof(Shared) + (size_t)a.per * sizeof(T);
  cudaError_t e = sg::allow_smem(k_sample<T>, smem, dev, allowed);
  if (e != cudaSuccess) return e;
  // Where a top-k is given and the GPU does not hold all clusters at once (two
  // CTAs on an SM), k_sample_rows goes first: 128256 fp32 logits under top-k 50
  // and top-p, 48 rows 22 us, 128 rows 33 us, against 28 and 67 with clusters
  // only; 32 rows 21 against 19. A row without a top-k is not its own, greedy
  // ones neither: one block would read all of it.
  a.pending = a.top_k && rows * cluster > 2 * sms;
  if (a.pending) {
    e = sg::try_launch(k_sample_rows<T>, dim3((unsigned)rows), dim3(kThreads), 0, 1, s, a);
    if (e != cudaSuccess) return e;
  }
  return sg::try_launch(k_sample<T>, dim3((unsigned)(rows * cluster)), dim3(kThreads), smem,
                        cluster, s, a);
}

}  // namespace

extern "C" int strasgpt_k_sample(const void* logits, int type, long long ld, int rows, int vocab,
                                 const float* temperature, const int* top_k, const float* top_p,
                                 const float* min_p, const float* u, int* token, float* prob,
                                 int* kept, void* stream) {
  const char* const me = "strasgpt_k_sample";
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return sg::refuse(me, "unknown type");
  if (rows < 0 || vocab <= 0) return sg::refuse(me, "empty shape");
  if (vocab > STRASGPT_SAMPLE_MAX_VOCAB) return sg::refuse(me, "vocabulary above 360448");
  if (rows > (1 << 24)) return sg::refuse(me, "too many rows");
  if (rows > 1 && ld < vocab) return sg::refuse(me, "rows of logits overlap");
  if (rows == 0) return 0;
  if (!logits || !u || !token) return sg::refuse(me, "null buffer");
  const size_t size = type == STRASGPT_F32 ? 4 : 2;
  if (!sg::aligned(logits, size)) return sg::refuse(me, "logits are not aligned to their entries");
  for (const void* p : {(const void*)temperature, (const void*)top_k, (const void*)top_p,
                        (const void*)min_p, (const void*)u, (const void*)token,
                        (const void*)prob, (const void*)kept})
    if (!sg::aligned(p, 4)) return sg::refuse(me, "a buffer is not aligned to its entries");
  // A token also says which kernel a row is left to, while filters are read.
  const void* const by_row[] = {token, prob, kept, temperature, top_k, top_p, min_p, u};
  for (int i = 0; i < 3; i++)
    for (int j = i + 1; j < 8; j++)
      if (by_row[i] && by_row[j] && sg::overlap(by_row[i], by_row[j], (size_t)rows * 4))
        return sg::refuse(me, "token, prob and kept must not share memory with each other or the "
                              "inputs");
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {logits, (const void*)temperature, (const void*)top_k, (const void*)top_p,
                        (const void*)min_p, (const void*)u, (const void*)token,
                        (const void*)prob, (const void*)kept})
    if (p)
      if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);

  // Eight CTAs a row; fewer for a small vocabulary, whose slices would cost
  // more in exchanges than they save in reading, and for as many rows as
  // still give every SM a CTA, as long as slices leave room for two on an SM
  // (128 rows of 32003 fp32 logits under top-p: 49 us with 2 a row, 113 us
  // with 8; 64 rows: 37 us with 4, 61 us with 8, 47 us with 2).
  int cluster = kMaxCluster;
  while (cluster > 1) {
    const int half = cluster / 2, slice = (vocab + half - 1) / half;
    const bool small = (vocab + cluster - 1) / cluster < 2048;
    if (!small && ((long long)rows * half < sms || slice * size > kSliceBytes)) break;
    cluster = half;
  }
  SampleArgs a;
  a.logits = logits; a.ld = ld; a.vocab = vocab;
  a.per = ((vocab + cluster - 1) / cluster + 7) & ~7;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u;
  a.token = token; a.prob = prob; a.kept = kept;
  a.vec = sg::aligned(logits, 16) && (rows == 1 || ld * size % 16 == 0);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = type == STRASGPT_F32 ? launch<float>(a, rows, cluster, sms, dev, s)
                                             : launch<uint16_t>(a, rows, cluster, sms, dev, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}
