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
// gather are integers, in a unit of 2^-42 of the largest weight that can be
// in their bin of the histogram, and all others are added in a fixed order:
// the same row gives the same bits whatever the order of CTAs and threads.
//
// A row is a thread-block cluster, each CTA holding a slice of it in shared
// memory: logits are read from HBM once, whatever the filters then need. No
// sort: one histogram over the logit's distance from M finds the bin in which
// a filter's border lies (a count for top-k, a mass for top-p); the entries
// of that bin, a few as a rule, are exchanged and ranked among themselves. A
// bin with more entries than kList is divided again, by key, until few or
// only equal ones are left.
#include <cooperative_groups.h>

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
constexpr int kBins = 1024;      // two per thread
constexpr int kList = 256;       // entries ranked against each other
constexpr int kUnit = 42;        // a weight in its bin's unit is at most 2^kUnit
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
};

struct Entry {
  unsigned key;
  int idx;
  u64 w;                         // in the bin's unit
};

// What a CTA's threads share, before its slice of the row.
struct alignas(16) Shared {
  double table[256];             // 2^(i / 256)
  u64 gmass[kBins];              // histogram of the row: mass, count
  unsigned gcount[kBins];
  unsigned count[kBins];         // of this slice: count, mass as two words
  unsigned lo[kBins], hi[kBins];
  Entry list[2][kList];          // border entries of top-k, of top-p
  // One slot per CTA of the cluster, written by that CTA in all of them.
  u64 best[kMaxCluster];
  float least[kMaxCluster];
  unsigned kmin[kMaxCluster], kmax[kMaxCluster];
  unsigned number[kMaxCluster];
  double mass[kMaxCluster];
  unsigned total[kMaxCluster];
  u64 wred[kWarps];
  double wsum[kWarps];
  unsigned wmin[kWarps], wmax[kWarps];
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
  N before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w == warp) before = all;
    all += red[w];
  }
  *total = all;
  return before + v;
}

// 2^e for -1022 <= e <= 1023.
__device__ __forceinline__ double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

template <typename T>
struct Row {
  Shared* sh;
  const T* xs;                   // this CTA's slice
  cg::cluster_group cluster;
  int rank, ranks;
  int start;                     // the slice's first index
  int c0, c1;                    // this thread's entries [c0, c1) of it
  float M;
  double scale;                  // log2(e) / T
  float bins_per;                // histogram bins per unit of logit

  __device__ float at(int i) const { return clean(load_f(xs[i])); }

  // exp((x - M) / T): 2^t with t in units of 1/256 taken apart by adding
  // 1.5 * 2^44, a cubic for the rest (|r ln 2| < 1.4e-3, the next term is
  // below 1.5e-13). 0 below 2^-1000.
  __device__ double weight(float x) const {
    if (x == M) return 1.0;
    const double t = ((double)x - (double)M) * scale;
    if (!(t > -1000.0)) return 0.0;      // also -inf, and NaN of M = inf
    const double magic = 6755399441055744.0 / 256;
    const double z = t + magic;
    const int n = __double2loint(z);
    const double r = (t - (z - magic)) * 0.6931471805599453;
    const double p = fma(fma(fma(r, 1.0 / 6, 0.5), r, 1.0), r, 1.0);
    return sh->table[n & 255] * p * pow2(n >> 8);
  }

  // Histogram bin, larger logits first; the last one is open to below.
  __device__ int bin_of(float x) const {
    if (x == M) return 0;
    return min(kBins - 1, (int)fminf((M - x) * bins_per, (float)kBins));
  }
  // The weights of bin b are at most 2^-e: their unit is 2^-(e + kUnit).
  __device__ int unit_of(int b) const {
    return kUnit + (int)fmin(b * (scale / (double)bins_per), 2.0 * kReach);
  }
  // A weight in units of 2^-unit, rounded: adding 2^52 leaves the nearest
  // integer in the low 52 bits. (A rounding of the bin's border may let a
  // weight exceed 2^kUnit by a little, not by 2^10.)
  __device__ u64 in_units(double w, int unit) const {
    return (u64)__double_as_longlong(fma(w, pow2(unit), 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }

  // The cluster's histogram of the entries that `digit` puts in [0, kBins);
  // unit(bin) is the unit of a bin's weights.
  template <typename F, typename G>
  __device__ void histogram(F digit, G unit) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh->count[b] = sh->lo[b] = sh->hi[b] = 0;
    __syncthreads();
    for (int i = c0; i < c1; i++) {
      const float x = at(i);
      const int b = digit(x);
      if (b < 0) continue;
      atomicAdd(&sh->count[b], 1u);
      const u64 w = in_units(weight(x), unit(b));
      if (w) {
        const unsigned l = (unsigned)w;
        const unsigned old = atomicAdd(&sh->lo[b], l);
        const unsigned h = (unsigned)(w >> 32) + (old + l < old);
        if (h) atomicAdd(&sh->hi[b], h);
      }
    }
    cluster.sync();
    // Each CTA adds up its share of the bins and hands it to all.
    const int share = kBins / ranks;
    for (int i = threadIdx.x; i < share; i += kThreads) {
      const int b = rank * share + i;
      unsigned c = 0;
      u64 m = 0;
      for (int r = 0; r < ranks; r++) {
        const Shared* o = cluster.map_shared_rank(sh, r);
        c += o->count[b];
        m += ((u64)o->hi[b] << 32) + o->lo[b];
      }
      for (int r = 0; r < ranks; r++) {
        Shared* o = cluster.map_shared_rank(sh, r);
        o->gcount[b] = c;
        o->gmass[b] = m;
      }
    }
    cluster.sync();
  }
  __device__ void histogram() {
    histogram([&](float x) { return x == -INFINITY ? -1 : bin_of(x); },
              [&](int b) { return unit_of(b); });
  }

  // The mass of a bin of the whole row's histogram.
  __device__ double mass_of(int b) const { return (double)sh->gmass[b] * pow2(-unit_of(b)); }

  // The row's mass, from its histogram.
  __device__ double mass() {
    double all;
    const int b = 2 * threadIdx.x;
    block_prefix(mass_of(b) + mass_of(b + 1), sh->wsum, &all);
    return all;
  }

  // The bin with the border: the first whose entries bring the count to k
  // (by_mass: the mass to target). Leaves it in sh->bbin, the count before it
  // in sh->bcount, the mass in sh->bbase (whole row) or, in units, in
  // sh->bmass (within a bin of it); false: no bin does.
  __device__ bool find_bin(bool by_mass, double target, unsigned k) {
    const int b = 2 * threadIdx.x;
    const unsigned c[2] = {sh->gcount[b], sh->gcount[b + 1]};
    const double m[2] = {mass_of(b), mass_of(b + 1)};
    u64 all;
    double mall;
    const unsigned upto = (unsigned)block_prefix((u64)(c[0] + c[1]), sh->wred, &all);
    const double mupto = block_prefix(m[0] + m[1], sh->wsum, &mall);
    if (threadIdx.x == 0) sh->bbin = kBins;
    __syncthreads();
    // A bin without entries is no border, whatever its sums' roundings say.
    const bool first = c[0] && (by_mass ? mupto - m[1] >= target : upto - c[1] >= k);
    const bool second = c[1] && (by_mass ? mupto >= target : upto >= k);
    if (first || second) atomicMin(&sh->bbin, (unsigned)(first ? b : b + 1));
    __syncthreads();
    const unsigned bin = sh->bbin;
    if ((bin >> 1) == threadIdx.x) {
      sh->bcount = upto - c[1] - (bin & 1 ? 0 : c[0]);
      sh->bbase = bin & 1 ? mupto - m[1] : mupto - m[1] - m[0];
    }
    __syncthreads();
    return bin < kBins;
  }

  // The same within one bin of the row's histogram: integers, on top of
  // `count`, `base` and `mass` before it.
  __device__ void find_sub_bin(bool by_mass, double target, unsigned k, unsigned count,
                               double base, u64 mass, double unit) {
    const int b = 2 * threadIdx.x;
    const unsigned c1_ = sh->gcount[b + 1], c0_ = sh->gcount[b];
    const u64 m1 = sh->gmass[b + 1], m0 = sh->gmass[b];
    u64 all;
    const unsigned upto = count + (unsigned)block_prefix((u64)(c0_ + c1_), sh->wred, &all);
    const u64 mupto = mass + block_prefix(m0 + m1, sh->wred, &all);
    if (threadIdx.x == 0) sh->bbin = kBins;
    __syncthreads();
    const bool first =
        c0_ && (by_mass ? base + (double)(mupto - m1) * unit >= target : upto - c1_ >= k);
    const bool second =
        c1_ && (by_mass ? base + (double)mupto * unit >= target : upto >= k);
    if (first || second) atomicMin(&sh->bbin, (unsigned)(first ? b : b + 1));
    __syncthreads();
    unsigned bin = sh->bbin;
    if (bin == kBins) {
      // Roundings of the row's sums left the border behind the bin's last
      // entry: that one it is.
      __syncthreads();
      if (threadIdx.x == 0) sh->bbin = 0;
      __syncthreads();
      if (c0_ || c1_) atomicMax(&sh->bbin, (unsigned)(c1_ ? b + 1 : b));
      __syncthreads();
      bin = sh->bbin;
    }
    if ((bin >> 1) == threadIdx.x) {
      sh->bcount = upto - c1_ - (bin & 1 ? 0 : c0_);
      sh->bmass = mupto - m1 - (bin & 1 ? 0 : m0);
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
      for (int i0 = a; i0 < b; i0 += 32) {
        const int i = i0 + lane;
        const double v = i < b ? value(at(i), start + i) : 0.0;
        double s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double n = shfl_up(s, o);
          if (lane >= o) s += n;
        }
        const unsigned some = __ballot_sync(0xFFFFFFFFu, v > 0);
        const unsigned over = __ballot_sync(0xFFFFFFFFu, v > 0 && run + s > target);
        if (some) last = i0 + 31 - __clz(some);
        if (over) {
          last = i0 + __ffs(over) - 1;
          break;
        }
        run += __shfl_sync(0xFFFFFFFFu, s, 31);
      }
      if (lane == 0) sh->found = last;
    }
    __syncthreads();
    return start + sh->found;
  }

  // The prefix of the order that a filter keeps: its last entry (key and
  // index) and, of top-k, its mass. tail: the border lies among entries of
  // weight 0; all others are kept, and `zeros` of those.
  struct Cut {
    unsigned key;
    int idx;
    double mass;
    bool tail;
    unsigned zeros;
  };

  // by_mass: the shortest prefix whose mass reaches `target`; else the first
  // k. ready: the row's histogram is there.
  __device__ Cut select(bool by_mass, double target, unsigned k, bool& ready, int which) {
    Cut cut = {0u, INT_MAX, 0.0, false, 0u};
    if (!ready) histogram();
    ready = true;
    if (!find_bin(by_mass, target, k)) {  // fewer than k entries: all are kept
      cut.mass = mass();
      return cut;
    }
    const int bin = (int)sh->bbin, unit = unit_of(bin);
    const double step = pow2(-unit), base = sh->bbase;
    unsigned count = sh->bcount, number = sh->gcount[bin];
    u64 mass = 0;                         // within the bin, before its border
    if (bin == kBins - 1 && sh->gmass[bin] == 0) {
      cut.tail = true;
      cut.zeros = k - count;
      cut.mass = base;
      return cut;
    }
    unsigned lo = 0, hi = 0xFFFFFFFFu;    // keys of the bin that are left
    int digit = bin;
    auto in_set = [&](float x) {
      if (x == -INFINITY || bin_of(x) != bin) return false;
      const unsigned key = key_of(x);
      return key >= lo && key <= hi;
    };
    while (number > kList) {
      unsigned kmin = 0xFFFFFFFFu, kmax = 0, mine = 0;
      for (int i = c0; i < c1; i++) {
        const float x = at(i);
        if (!in_set(x)) continue;
        mine++;
        const unsigned key = key_of(x);
        kmin = min(kmin, key);
        kmax = max(kmax, key);
      }
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
        const u64 w = in_units(weight(of_key(kmin)), unit);
        unsigned take = by_mass ? number : k - count;
        if (by_mass && w > 0) {
          const double need = (target - (base + (double)mass * step)) / ((double)w * step);
          if (need < (double)number) take = need > 1.0 ? (unsigned)ceil(need) : 1u;
        }
        cut.key = kmin;
        cut.mass = base + (double)(mass + take * w) * step;
        if (take < number) {
          // The take-th of them lies in one slice.
          if (before < take && take <= before + (unsigned)total) {
            const int i = find_index([&](float x, int) { return in_set(x) ? 1.0 : 0.0; },
                                     (double)mine, upto, (double)(take - 1 - before));
            if (threadIdx.x < ranks) cluster.map_shared_rank(sh, threadIdx.x)->cut_idx = i;
          }
          cluster.sync();
          cut.idx = sh->cut_idx;
        }
        return cut;
      }
      int shift = 0;
      while (((kmax - kmin) >> shift) >= (unsigned)kBins) shift++;
      lo = kmin;
      hi = kmax;
      histogram([&](float x) { return in_set(x) ? (int)((kmax - key_of(x)) >> shift) : -1; },
                [&](int) { return unit; });
      ready = false;
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
    if (threadIdx.x == 0) {
      unsigned before = 0;
      for (int r = 0; r < rank; r++) before += cluster.map_shared_rank(sh, r)->count[digit];
      sh->fill = before;
    }
    __syncthreads();
    for (int i = c0; i < c1; i++) {
      const float x = at(i);
      if (!in_set(x)) continue;
      const unsigned p = atomicAdd(&sh->fill, 1u);
      const Entry e = {key_of(x), start + i, in_units(weight(x), unit)};
      for (int r = 0; r < ranks; r++) cluster.map_shared_rank(sh, r)->list[which][p] = e;
    }
    cluster.sync();
    bool kept = false;
    unsigned place = 0;
    u64 ahead = mass;
    Entry e = {0u, 0, 0ull};
    if (threadIdx.x < number) {
      e = sh->list[which][threadIdx.x];
      for (unsigned j = 0; j < number; j++) {
        const Entry o = sh->list[which][j];
        if (o.key > e.key || (o.key == e.key && o.idx < e.idx)) {
          place++;
          ahead += o.w;
        }
      }
      // The border is in this set: its first entry is kept.
      kept = place == 0 ||
             (by_mass ? base + (double)ahead * step < target : count + place < k);
    }
    const unsigned keeps = __syncthreads_count(kept);
    if (kept && place == keeps - 1) {
      sh->cut_key = e.key;
      sh->cut_idx = e.idx;
      sh->bmass = ahead + e.w;
    }
    __syncthreads();
    cut.key = sh->cut_key;
    cut.idx = sh->cut_idx;
    cut.mass = base + (double)sh->bmass * step;
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
  if (threadIdx.x < 256) sh->table[threadIdx.x] = exp2(threadIdx.x / 256.0);
  sg::pdl_trigger();
  sg::pdl_wait();

  const int start = min(rank * a.per, a.vocab), n = min(a.per, a.vocab - start);
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + start;
  // Slice into shared memory; its largest key (with the lowest index that has
  // it) and its smallest finite logit.
  u64 best = 0;
  float least = INFINITY;
  auto take = [&](float x, int i) {
    const u64 b = ((u64)key_of(x) << 32) | (unsigned)(0x7FFFFFFF - (start + i));
    if (x > -INFINITY) {
      best = b > best ? b : best;
      least = fminf(least, x);
    }
  };
  constexpr int V = 16 / sizeof(T);
  const int nv = a.vec ? n / V : 0;
#pragma unroll 4
  for (int v = threadIdx.x; v < nv; v += kThreads) {
    const uint4 r = sg::ldg_stream(src + v * V);
    T e[V];
    memcpy(e, &r, 16);
#pragma unroll
    for (int j = 0; j < V; j++) take(clean(load_f(e[j])), v * V + j);
    reinterpret_cast<uint4*>(xs)[v] = r;
  }
  for (int i = nv * V + threadIdx.x; i < n; i += kThreads) {
    xs[i] = src[i];
    take(clean(load_f(xs[i])), i);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 b = __shfl_xor_sync(0xFFFFFFFFu, best, o);
    best = b > best ? b : best;
    least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
  }
  if (lane == 0) {
    sh->wred[warp] = best;
    sh->wmin[warp] = __float_as_uint(least);
  }
  __syncthreads();
  cluster.sync();  // every CTA of the cluster runs: its shared memory is there
  if (threadIdx.x < ranks) {
    for (int w = 0; w < kWarps; w++) {
      best = sh->wred[w] > best ? sh->wred[w] : best;
      least = fminf(least, __uint_as_float(sh->wmin[w]));
    }
    Shared* o = cluster.map_shared_rank(sh, threadIdx.x);
    o->best[rank] = best;
    o->least[rank] = least;
  }
  const float T_ = a.temperature ? a.temperature[row] : 1.f;
  const int k_ = a.top_k ? a.top_k[row] : 0;
  const float p_ = a.top_p ? a.top_p[row] : 1.f;
  const float m_ = a.min_p ? a.min_p[row] : 0.f;
  const float u_ = a.u[row];
  cluster.sync();
  best = 0;
  least = INFINITY;
  for (int r = 0; r < ranks; r++) {
    best = sh->best[r] > best ? sh->best[r] : best;
    least = fminf(least, sh->least[r]);
  }
  const bool empty = best == 0;
  if (empty || !(T_ > 0.f) || k_ == 1 || p_ <= 0.f) {
    if (rank == 0 && threadIdx.x == 0) {
      a.token[row] = empty ? -1 : 0x7FFFFFFF - (int)(unsigned)best;
      if (a.prob) a.prob[row] = empty ? 0.f : 1.f;
      if (a.kept) a.kept[row] = empty ? 0 : 1;
    }
    return;
  }

  const int chunk = ((a.per + kThreads - 1) / kThreads) | 1;  // odd: no bank conflicts
  Row<T> r{sh, xs, cluster, rank, ranks, start};
  r.c0 = min((int)threadIdx.x * chunk, n);
  r.c1 = min(r.c0 + chunk, n);
  r.M = of_key((unsigned)(best >> 32));
  r.scale = 1.4426950408889634 / (double)T_;
  // The bins share what is within kReach octaves of the largest weight, or
  // down to the smallest logit if that is nearer.
  double range = fmin(kReach / r.scale, ((double)r.M - (double)least) * (1 + 1e-6));
  if (!(range < 1e300)) range = 1;  // infinite logits at an infinite temperature
  r.bins_per = (float)((kBins - 1) / range);
  const double min_w = m_ > 0.f ? fmin((double)m_, 1.0) : 0.0;

  typename Row<T>::Cut cut = {0u, INT_MAX, 0.0, false, 0u};
  bool ready = false, cut_k = false;
  if (k_ > 1 && k_ < a.vocab) {
    cut = r.select(false, 0.0, (unsigned)k_, ready, 0);
    cut_k = true;
  }
  if (p_ < 1.f) {
    if (!cut_k) {
      r.histogram();
      ready = true;
      cut.mass = r.mass();
    }
    cut = r.select(true, (double)p_ * cut.mass, 0u, ready, 1);
  }

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
  double mine = 0;
  int number = 0;
  for (int i = r.c0; i < r.c1; i++) {
    bool kept;
    mine += kept_weight(r.at(i), start + i, kept);
    number += kept;
  }
  double total;
  u64 numbers;
  const double upto = block_prefix(mine, sh->wsum, &total);
  block_prefix((u64)number, sh->wred, &numbers);
  if (threadIdx.x < ranks) {
    Shared* o = cluster.map_shared_rank(sh, threadIdx.x);
    o->mass[rank] = total;
    o->total[rank] = (unsigned)numbers;
  }
  cluster.sync();
  total = 0;
  unsigned kept = 0;
  for (int q = 0; q < ranks; q++) {
    total += sh->mass[q];
    kept += sh->total[q];
  }
  // The slice in which the running mass exceeds u total; the last with any
  // if none (u at or above 1).
  const double target = u_ > 0.f ? (double)u_ * total : 0.0;
  double run = 0, before = 0;
  int owner = -1;
  for (int q = 0; q < ranks; q++) {
    const double v = sh->mass[q];
    if (v > 0 && (owner < 0 || !(run > target))) {
      owner = q;
      before = run;
    }
    run += v;
  }
  if (rank != owner) return;
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

template <typename T>
cudaError_t launch(const SampleArgs& a, int rows, int cluster, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  const size_t smem = sizeof(Shared) + (size_t)a.per * sizeof(T);
  const cudaError_t e = sg::allow_smem(k_sample<T>, smem, dev, allowed);
  if (e != cudaSuccess) return e;
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
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {logits, (const void*)temperature, (const void*)top_k, (const void*)top_p,
                        (const void*)min_p, (const void*)u, (const void*)token,
                        (const void*)prob, (const void*)kept})
    if (p)
      if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);

  // Eight CTAs a row; fewer for a small vocabulary, whose slices would cost
  // more in exchanges than they save in reading.
  int cluster = kMaxCluster;
  while (cluster > 1 && (vocab + cluster - 1) / cluster < 2048) cluster /= 2;
  SampleArgs a;
  a.logits = logits; a.ld = ld; a.vocab = vocab;
  a.per = ((vocab + cluster - 1) / cluster + 7) & ~7;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u;
  a.token = token; a.prob = prob; a.kept = kept;
  a.vec = sg::aligned(logits, 16) && (rows == 1 || ld * size % 16 == 0);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = type == STRASGPT_F32 ? launch<float>(a, rows, cluster, dev, s)
                                             : launch<uint16_t>(a, rows, cluster, dev, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}
