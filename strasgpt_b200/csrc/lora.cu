// strasgpt_k_lora: low-rank adapters of many requests at once, beside a
// projection that all of them share.
//
// Token i with adapter d adds scale_d B_d (A_d x_i) to its row of the shared
// projection. Per token that is two thin products, k entries down to `rank`
// and up to n: with ranks of 8 to 128, bytes are what it costs, x and the
// projection's rows for many tokens, the adapters themselves for single ones.
//
// One launch, no workspace: a cluster of CTAs takes a tile of tokens. Each CTA
// multiplies its share of the k entries with A, the cluster's CTAs add up their
// sums over distributed shared memory (in a fixed order, and each sends what
// the others need, so that no load waits on another SM), and each CTA then has
// its share of the n outputs: base, products with B, epilogue.
//
// Tokens are the rows of mma.sync.m16n8k16 (16 of them; tcgen05's 128 would
// be empty for single tokens, and the products are not what bounds this). A
// block of 16 rows is multiplied once for each adapter in it, and every row
// keeps its own adapter's sums: whatever another adapter's weights hold stays
// out of it. Runs of tokens of one adapter cost one product, 16 single tokens
// of a batch read the weights they would read anyway.
//
// Operands go from global memory to registers: the order of a product's k
// entries is free as long as both operands have the same, so that a lane's
// entries of a fragment are 16 (x: 32) consecutive bytes.
//
// Precision: fp32 rows are three bf16 parts of 8 bits, all 24 of them, and the
// weights are bf16, so products are exact; the tensor cores cut their sums,
// which are therefore taken from zero for 32 entries at a time (small parts
// first) and added with rounding. A x is held in 32 bits, as three parts (fp32
// rows) or two (bf16 rows: 2^-17 of it, where the result has 2^-9).
#include "entry.h"

#include <limits.h>

#include <algorithm>

extern "C" {
#include "strasgpt_kernels.h"
}

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kCluster = 8;     // CTAs of a tile of tokens
constexpr int kMaxTokens = 64;  // of a tile
constexpr int kDirect = 1024;   // sums of a tile that every CTA adds up for itself

struct LoraArgs {
  const void* x;
  const uint16_t *a, *b;
  const void* base;
  void* out;
  const int* adapter;
  const float* scale;
  long long ldx, ldb, ldo;
  int m, k, n, rank, adapters;
  int tokens;   // of a tile
  int epi;
  bool wide;    // base and out rows in 16-byte (out of SwiGLU: half as wide) accesses
};

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The upper halves of two words: two values cut to bf16.
__device__ __forceinline__ uint32_t upper(float x0, float x1) {
  return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}
__device__ __forceinline__ float rest(float x) {  // what the cut leaves, exact
  return x - __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t bf16x2(float x0, float x1) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(x1), "f"(x0));
  return w;
}
// Two values as N bf16 parts: 3 lose nothing, the second of 2 is rounded. An
// infinity is one in the first part, and NaN in the others.
template <int N>
__device__ __forceinline__ void parts(float x0, float x1, uint32_t* p, int step) {
  p[0] = upper(x0, x1);
  x0 = rest(x0);
  x1 = rest(x1);
  if constexpr (N == 2) {
    p[step] = bf16x2(x0, x1);
  } else {
    p[step] = upper(x0, x1);
    p[2 * step] = upper(rest(x0), rest(x1));
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Stores v to p's place in the shared memory of the cluster's CTA `to`.
__device__ __forceinline__ void store_to(const float* p, uint32_t to, float v) {
  asm volatile(
      "{\n .reg .u32 at;\n mapa.shared::cluster.u32 at, %0, %1;\n"
      " st.shared::cluster.f32 [at], %2;\n}" ::"r"((uint32_t)__cvta_generic_to_shared(p)),
      "r"(to), "f"(v)
      : "memory");
}

// N neighbouring results, rounded once.
template <int N>
__device__ __forceinline__ void store(float* to, const float* v, int count, bool wide) {
  if (wide && count == N) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < count) to[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void store(uint16_t* to, const float* v, int count, bool wide) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; i++) w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
  if (wide && count == N) {
    if constexpr (N == 8)
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < count) to[i] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
  }
}
// N neighbouring values, zeros behind the last.
template <int N>
__device__ __forceinline__ void load(const float* from, float* v, int count, bool wide) {
  if (wide && count == N) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(from + i);
      v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < count ? from[i] : 0.f;
  }
}
template <int N>
__device__ __forceinline__ void load(const uint16_t* from, float* v, int count, bool wide) {
  if (wide && count == N) {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(from);
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(from);
      w[0] = x.x; w[1] = x.y;
    }
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      v[2 * i] = sg::bf16_lo(w[i]);
      v[2 * i + 1] = sg::bf16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < count ? sg::bf16_to_f32(from[i]) : 0.f;
  }
}

// MW blocks of 16 tokens; the warps of a block share out its k entries, then
// its outputs. Ranks up to 8 RN.
template <int MW, int RN>
struct Shape {
  static constexpr int kKW = kWarps / MW;
  static constexpr int kRow = 8 * RN + 4;  // floats of a row of sums: no bank twice
  static constexpr int kSums = kWarps * 16 * kRow;      // [kKW][16 MW][kRow]
  static constexpr size_t bytes(int tokens, int rank) {
    return sizeof(float) * (kSums + (tokens * rank <= kDirect ? kCluster : 1) * tokens * rank);
  }
};

template <typename T, int MW, int RN>
__global__ void __launch_bounds__(kThreads, RN > 2 ? 2 : 3) k_lora(const LoraArgs p) {
  using S = Shape<MW, RN>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kKW = S::kKW, kRow = S::kRow;
  constexpr int kXParts = kF32 ? 3 : 1, kSParts = kF32 ? 3 : 2;
  extern __shared__ __align__(16) float smem[];
  __shared__ int ids[kMaxTokens];
  float* const sums = smem;
  float* const exchange = smem + S::kSums;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
  const int mw = warp % MW, kw = warp / MW;
  const uint32_t cta = cluster_rank();
  const int t0 = blockIdx.x / kCluster * p.tokens, nt = min(p.tokens, p.m - t0);
  sg::pdl_trigger();
  sg::pdl_wait();
  if (threadIdx.x < kMaxTokens) {
    const int id = threadIdx.x < nt ? p.adapter[t0 + threadIdx.x] : -1;
    ids[threadIdx.x] = id >= 0 && id < p.adapters ? id : -1;
  }
  __syncthreads();
  // This lane's rows of the block, and the adapter of row lane % 16.
  const int rA = 16 * mw + g8, rB = rA + 8;
  const int idA = ids[rA], idB = ids[rB], mine = ids[16 * mw + (lane & 15)];

  // --- A x: this CTA's steps of 32 entries, taken in turn by the block's warps.
  const int steps = (p.k + 31) / 32, per = (steps + kCluster - 1) / kCluster;
  const int step0 = cta * per, step1 = min(steps, step0 + per);
  const T* const xA = static_cast<const T*>(p.x) + (size_t)(t0 + (idA >= 0 ? rA : 0)) * p.ldx;
  const T* const xB = static_cast<const T*>(p.x) + (size_t)(t0 + (idB >= 0 ? rB : 0)) * p.ldx;
  for (unsigned left = __ballot_sync(0xFFFFFFFFu, mine >= 0) & 0xFFFFu; left;) {
    const int d = __shfl_sync(0xFFFFFFFFu, mine, __ffs(left) - 1);
    left &= ~__ballot_sync(0xFFFFFFFFu, mine == d);
    const uint16_t* const w = p.a + (size_t)d * p.rank * p.k;
    float acc[RN][4];
#pragma unroll
    for (int j = 0; j < RN; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 2
    for (int s = step0 + kw; s < step1; s += kKW) {
      const int k0 = 32 * s + 8 * c4;
      const bool in = k0 < p.k;
      // Rows of other adapters are zeros: they are not kept.
      uint32_t xa[2][kXParts][4];
      if constexpr (kF32) {
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        float4 v[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          v[0][h] = in && idA == d ? *reinterpret_cast<const float4*>(xA + k0 + 4 * h) : zero;
          v[1][h] = in && idB == d ? *reinterpret_cast<const float4*>(xB + k0 + 4 * h) : zero;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          parts<3>(v[0][h].x, v[0][h].y, &xa[h][0][0], 4);
          parts<3>(v[1][h].x, v[1][h].y, &xa[h][0][1], 4);
          parts<3>(v[0][h].z, v[0][h].w, &xa[h][0][2], 4);
          parts<3>(v[1][h].z, v[1][h].w, &xa[h][0][3], 4);
        }
      } else {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 v = in && idA == d ? *reinterpret_cast<const uint4*>(xA + k0) : zero;
        const uint4 z = in && idB == d ? *reinterpret_cast<const uint4*>(xB + k0) : zero;
        xa[0][0][0] = v.x; xa[0][0][1] = z.x; xa[0][0][2] = v.y; xa[0][0][3] = z.y;
        xa[1][0][0] = v.z; xa[1][0][1] = z.z; xa[1][0][2] = v.w; xa[1][0][3] = z.w;
      }
#pragma unroll
      for (int j = 0; j < RN; j++) {
        if (8 * j >= p.rank) break;
        const uint4 b = in ? *reinterpret_cast<const uint4*>(w + (size_t)(8 * j + g8) * p.k + k0)
                           : make_uint4(0, 0, 0, 0);
        if constexpr (kF32) {
          float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 2; q >= 0; q--) {
            mma_bf16(y, xa[0][q], b.x, b.y);
            mma_bf16(y, xa[1][q], b.z, b.w);
          }
#pragma unroll
          for (int e = 0; e < 4; e++) acc[j][e] += y[e];
        } else {
          mma_bf16(acc[j], xa[0][0], b.x, b.y);
          mma_bf16(acc[j], xa[1][0], b.z, b.w);
        }
      }
    }
    float* const to = sums + kw * 16 * MW * kRow;
#pragma unroll
    for (int j = 0; j < RN; j++) {
      if (8 * j >= p.rank) break;
      if (idA == d) *reinterpret_cast<float2*>(to + rA * kRow + 8 * j + 2 * c4) =
          make_float2(acc[j][0], acc[j][1]);
      if (idB == d) *reinterpret_cast<float2*>(to + rB * kRow + 8 * j + 2 * c4) =
          make_float2(acc[j][2], acc[j][3]);
    }
  }
  __syncthreads();

  // --- The cluster's sums. Entry e is of row e / rank. (Rows without an adapter
  // have whatever lies there: they are not used.)
  const int every = p.tokens * p.rank;
  auto warps = [&](int e) {
    const float* from = sums + e / p.rank * kRow + e % p.rank;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kKW; w++) v += from[w * 16 * MW * kRow];
    return v;
  };
  auto ctas = [&](const float* from, int step) {
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kCluster; c++) v += from[c * step];
    return v;
  };
  auto scale = [&](int e) {
    const int id = ids[e / p.rank];
    return p.scale && id >= 0 ? p.scale[id] : 1.f;
  };
  if (every <= kDirect) {
    for (int e = threadIdx.x; e < every; e += kThreads) {
      const float v = warps(e);
#pragma unroll
      for (uint32_t c = 0; c < kCluster; c++) store_to(exchange + cta * every + e, c, v);
    }
    cluster_sync();
    for (int e = threadIdx.x; e < every; e += kThreads)
      sums[e / p.rank * kRow + e % p.rank] = ctas(exchange + e, every) * scale(e);
  } else {
    const int slice = every / kCluster;  // rank is a multiple of 8
    for (int e = threadIdx.x; e < every; e += kThreads)
      store_to(exchange + cta * slice + e % slice, e / slice, warps(e));
    cluster_sync();
    for (int i = threadIdx.x; i < slice; i += kThreads) {
      const int e = cta * slice + i;
      const float v = ctas(exchange + i, slice) * scale(e);
#pragma unroll
      for (uint32_t c = 0; c < kCluster; c++) store_to(sums + e / p.rank * kRow + e % p.rank, c, v);
    }
    cluster_sync();
  }
  __syncthreads();

  // --- B (A x): the sums as fragments, 16 ranks a step, lane c4 having four of
  // them in a row.
  constexpr int kSteps = (RN + 1) / 2;
  uint32_t sa[kSteps][kSParts][4];
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int r0 = 16 * u + 4 * c4;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 v = r0 < p.rank && idA >= 0
                         ? *reinterpret_cast<const float4*>(sums + rA * kRow + r0) : zero;
    const float4 z = r0 < p.rank && idB >= 0
                         ? *reinterpret_cast<const float4*>(sums + rB * kRow + r0) : zero;
    parts<kSParts>(v.x, v.y, &sa[u][0][0], 4);
    parts<kSParts>(z.x, z.y, &sa[u][0][1], 4);
    parts<kSParts>(v.z, v.w, &sa[u][0][2], 4);
    parts<kSParts>(z.z, z.w, &sa[u][0][3], 4);
  }
  // Tiles of 32 outputs, four products wide: column q of product j is output
  // 8 (q / 2) + 2 j + q % 2, so that a lane has outputs 8 c4 to 8 c4 + 7 of two
  // tokens.
  const int tiles = (p.n + 31) / 32, share = (tiles + kCluster - 1) / kCluster;
  const int tile1 = min(tiles, (int)(cta + 1) * share);
  const bool inA = rA < nt, inB = rB < nt;
  const size_t tA = t0 + (inA ? rA : 0), tB = t0 + (inB ? rB : 0);
  const T* const baseA = static_cast<const T*>(p.base) + tA * p.ldb;
  const T* const baseB = static_cast<const T*>(p.base) + tB * p.ldb;
  for (int tile = cta * share + kw; tile < tile1; tile += kKW) {
    const int n0 = 32 * tile + 8 * c4, count = max(0, min(8, p.n - n0));
    float vA[8], vB[8];
    load<8>(baseA + n0, vA, inA && p.base ? count : 0, p.wide);
    load<8>(baseB + n0, vB, inB && p.base ? count : 0, p.wide);
    const int row0 = 32 * tile + 8 * (g8 >> 1) + (g8 & 1);  // B's row of product 0
    for (unsigned left = __ballot_sync(0xFFFFFFFFu, mine >= 0) & 0xFFFFu; left;) {
      const int d = __shfl_sync(0xFFFFFFFFu, mine, __ffs(left) - 1);
      left &= ~__ballot_sync(0xFFFFFFFFu, mine == d);
      const uint16_t* const w = p.b + (size_t)d * p.n * p.rank;
      float big[4][4], small[4][4];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) big[j][e] = small[j][e] = 0.f;
#pragma unroll
      for (int u = 0; u < kSteps; u++) {
        const int r0 = 16 * u + 4 * c4;
        if (16 * u >= p.rank) break;
        uint2 b[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
          b[j] = r0 < p.rank && row0 + 2 * j < p.n
                     ? *reinterpret_cast<const uint2*>(w + (size_t)(row0 + 2 * j) * p.rank + r0)
                     : make_uint2(0, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
          for (int q = kSParts - 1; q > 0; q--) mma_bf16(small[j], sa[u][q], b[j].x, b[j].y);
          mma_bf16(big[j], sa[u][0], b[j].x, b[j].y);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          if (idA == d) vA[2 * j + e] += big[j][e] + small[j][e];
          if (idB == d) vB[2 * j + e] += big[j][2 + e] + small[j][2 + e];
        }
    }
    auto finish = [&](float* v, size_t token) {
      T* const row = static_cast<T*>(p.out) + token * p.ldo;
      if (p.epi == STRASGPT_EPI_SWIGLU) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = sg::swiglu(v[2 * i], v[2 * i + 1]);
        store<4>(row + n0 / 2, y, count / 2, p.wide);
      } else {
        if (p.epi == STRASGPT_EPI_ADD) {
          float old[8];
          load<8>(row + n0, old, count, p.wide);
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] += old[i];
        }
        store<8>(row + n0, v, count, p.wide);
      }
    };
    if (inA) finish(vA, tA);
    if (inB) finish(vB, tB);
  }
}

template <typename T, int MW, int RN>
cudaError_t launch(const LoraArgs& p, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  const size_t bytes = Shape<MW, RN>::bytes(p.tokens, p.rank);
  const cudaError_t e = sg::allow_smem(k_lora<T, MW, RN>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  const long long tiles = ((long long)p.m + p.tokens - 1) / p.tokens;
  return sg::try_launch(k_lora<T, MW, RN>, dim3((unsigned)(tiles * kCluster)), dim3(kThreads), bytes,
                        kCluster, s, p);
}

template <typename T, int MW>
cudaError_t launch_rank(const LoraArgs& p, int dev, cudaStream_t s) {
  if (p.rank <= 16) return launch<T, MW, 2>(p, dev, s);
  if (p.rank <= 32) return launch<T, MW, 4>(p, dev, s);
  if (p.rank <= 64) return launch<T, MW, 8>(p, dev, s);
  return launch<T, MW, 16>(p, dev, s);
}

template <typename T>
cudaError_t launch_type(const LoraArgs& p, int dev, cudaStream_t s) {
  if (p.tokens <= 16) return launch_rank<T, 1>(p, dev, s);
  if (p.tokens <= 32) return launch_rank<T, 2>(p, dev, s);
  return launch_rank<T, 4>(p, dev, s);
}

// Tokens of a tile: as few as leave no more than four CTAs to an SM.
int tokens_of(int m, int sms) {
  int t = 1;
  while (t < kMaxTokens && ((long long)m + t - 1) / t * kCluster > 4ll * sms) t *= 2;
  return t;
}

}  // namespace

extern "C" int strasgpt_k_lora(const void* x, long long ldx, const uint16_t* a, const uint16_t* b,
                               int type, int m, int k, int n, int rank, int adapters,
                               const int* adapter, const float* scale, const void* base,
                               long long ldb, void* out, long long ldo, int epi, void* stream) {
  const char* const me = "strasgpt_k_lora";
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return sg::refuse(me, "unknown type");
  if (m < 0 || k <= 0 || n <= 0 || adapters <= 0) return sg::refuse(me, "empty shape");
  if (rank < 8 || rank > STRASGPT_LORA_MAX_RANK || rank % 8)
    return sg::refuse(me, "rank must be a multiple of 8, 8 to 128");
  if (k % 8) return sg::refuse(me, "k must be a multiple of 8");
  if (epi != STRASGPT_EPI_STORE && epi != STRASGPT_EPI_ADD && epi != STRASGPT_EPI_SWIGLU)
    return sg::refuse(me, "unknown epilogue");
  const bool gated = epi == STRASGPT_EPI_SWIGLU;
  if (gated && n % 2) return sg::refuse(me, "odd swiglu rows");
  const int outs = gated ? n / 2 : n;
  if (m > 1 && (ldx < k || ldo < outs || (base && ldb < n)))
    return sg::refuse(me, "rows of x, base or out overlap");
  if (m == 0) return 0;
  if (!x || !a || !b || !adapter || !out) return sg::refuse(me, "null buffer");
  const size_t size = type == STRASGPT_F32 ? 4 : 2;
  if (!sg::aligned(x, 16) || !sg::aligned(a, 16) || !sg::aligned(b, 16) ||
      (m > 1 && ldx * size % 16))
    return sg::refuse(me, "x, its rows, a and b must be 16-byte aligned");
  if (!sg::aligned(base, size) || !sg::aligned(out, size) || !sg::aligned(adapter, 4) ||
      !sg::aligned(scale, 4))
    return sg::refuse(me, "a buffer is not aligned to its entries");
  if (x == out) return sg::refuse(me, "x cannot be out");
  if (base == out && (epi != STRASGPT_EPI_STORE || (m > 1 && ldb != ldo)))
    return sg::refuse(me, "base can be out only to be stored to, with the same stride");
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {x, (const void*)a, (const void*)b, (const void*)adapter,
                        (const void*)scale, base, (const void*)out})
    if (p)
      if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);
  LoraArgs p;
  p.x = x; p.a = a; p.b = b; p.base = base; p.out = out;
  p.adapter = adapter; p.scale = scale;
  p.ldx = ldx; p.ldb = base ? ldb : 0; p.ldo = ldo;
  p.m = m; p.k = k; p.n = n; p.rank = rank; p.adapters = adapters;
  p.epi = epi;
  const size_t step = gated ? 4 * size : 16;  // bytes of an access to out
  p.wide = sg::aligned(base, 16) && sg::aligned(out, step) &&
           (m == 1 || (p.ldb * size % 16 == 0 && ldo * size % step == 0));
  p.tokens = tokens_of(m, sms);
  const long long tiles = ((long long)m + p.tokens - 1) / p.tokens;
  if (tiles > INT_MAX / kCluster) return sg::refuse(me, "too many tokens");
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = type == STRASGPT_F32 ? launch_type<float>(p, dev, s)
                                             : launch_type<uint16_t>(p, dev, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}
