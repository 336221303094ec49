// strasgpt_k_lora: low-rank adapters of many requests at once, beside a
// projection that all of them share.
//
// Token i with adapter d adds scale_d B_d (A_d x_i) to its row of the shared
// projection. Per token that is two thin products, k entries down to `rank`
// and up to n: with ranks of 8 to 128, bytes are what it costs, x and the
// projection's rows for many tokens, the adapters themselves for single ones.
//
// One launch, no workspace: a cluster of eight CTAs (four where there are enough
// others) takes some tokens of one adapter. Each CTA multiplies its share of the k
// entries with A, the cluster adds up the sums over distributed shared memory, in a
// fixed order, and each CTA then has its share of the n outputs: base, products
// with B, epilogue. No product takes more than one adapter's tokens, and a product's
// rows, or columns, are tokens: whatever other adapters or tokens hold stays out.
//
// Two kernels. Up to kFew tokens, which may each have an adapter of their own:
// mma.sync with the weights as rows and up to eight tokens as columns, operands from
// global memory to registers (tcgen05's 128 rows and its hand-overs cost more than
// the weights' bytes). More: tcgen05 with the tokens as rows, all memory by TMA.
//
// Precision: fp32 rows are three bf16 parts of 8 bits, all 24 of them, and the
// weights are bf16, so products are exact; the tensor cores cut their sums, which
// are therefore taken from zero for 32 entries at a time, or kept apart for the large
// parts and the small ones, and added with rounding. A x is held in 32 bits, and is
// three parts (fp32 rows) or two (bf16 rows: 2^-17 of it, where the result has 2^-9).
//
// Measured on a B200, captured calls in short runs: 3.8 us for one token of 2048 x 2048,
// rank 8; 7.7 us for 61 tokens, most with one of 48 adapters of rank 16, on 4096 x 6144
// (latency: a read of A, the cluster's sums and a read of B, one after the other); 44 us
// for 2047 fp32 tokens of six prompts, rank 32, on 4096 x 4096 (2.4 TB/s); 144 us for 4001
// bf16 tokens, rank 64, on 4096 x 28672 with SwiGLU (2.8 TB/s). What bounds the last two is
// noted at k_lora_many.
#include "entry.h"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <limits.h>

#include <algorithm>

extern "C" {
#include "strasgpt_kernels.h"
}

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kCluster = 8;     // CTAs of a tile of tokens
constexpr int kMaxTokens = 128;  // of a tile

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
  bool base_tma, out_tma;  // what is added, out: TMA can read, write it
  bool wide;    // base and out rows: four entries (out of SwiGLU: two) are one access
};

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
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
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
// This CTA has started: the others may write to its shared memory.
__device__ __forceinline__ void cluster_started() {
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// Stores v to p's place in the shared memory of the cluster's CTA `to`.
__device__ __forceinline__ void store_to(const float* p, uint32_t to, float v) {
  asm volatile(
      "{\n .reg .u32 at;\n mapa.shared::cluster.u32 at, %0, %1;\n"
      " st.shared::cluster.f32 [at], %2;\n}" ::"r"((uint32_t)__cvta_generic_to_shared(p)),
      "r"(to), "f"(v)
      : "memory");
}

// One access.
template <int N>
struct alignas(N * 4) Words {
  uint32_t w[N];
};
__device__ __forceinline__ void store4_to(const float* p, uint32_t to, float4 v) {
  asm volatile(
      "{\n .reg .u32 at;\n mapa.shared::cluster.u32 at, %0, %1;\n"
      " st.shared::cluster.v4.f32 [at], {%2, %3, %4, %5};\n}" ::"r"(
          (uint32_t)__cvta_generic_to_shared(p)),
      "r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
      : "memory");
}
__device__ __forceinline__ float4 load4_from(const float* p, uint32_t from) {
  float4 v;
  asm volatile(
      "{\n .reg .u32 at;\n mapa.shared::cluster.u32 at, %4, %5;\n"
      " ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [at];\n}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(from)
      : "memory");
  return v;
}
// N neighbouring results (2, 4 or 8), rounded once.
template <int N>
__device__ __forceinline__ void store(float* to, const float* v, int count, bool wide) {
  if (wide && count == N) {
    constexpr int kW = N < 4 ? N : 4;
#pragma unroll
    for (int i = 0; i < N; i += kW) {
      Words<kW> x;
#pragma unroll
      for (int j = 0; j < kW; j++) x.w[j] = __float_as_uint(v[i + j]);
      *reinterpret_cast<Words<kW>*>(to + i) = x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < count) to[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void store(uint16_t* to, const float* v, int count, bool wide) {
  Words<N / 2> x;
#pragma unroll
  for (int i = 0; i < N / 2; i++) x.w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
  if (wide && count == N) {
    *reinterpret_cast<Words<N / 2>*>(to) = x;
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < count) to[i] = (uint16_t)(x.w[i / 2] >> (i % 2 * 16));
  }
}
// N neighbouring values (4 or 8), zeros behind the last.
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
    const Words<N / 2> x = *reinterpret_cast<const Words<N / 2>*>(from);
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      v[2 * i] = sg::bf16_lo(x.w[i]);
      v[2 * i + 1] = sg::bf16_hi(x.w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < count ? sg::bf16_to_f32(from[i]) : 0.f;
  }
}

// silu(gate) up. For results that are rounded to bf16, approximate exp and reciprocal:
// 2^-19 of the result for gates of up to 10, 2^-16 at -95.
__device__ __forceinline__ float swiglu(float gate, float up, float) {
  return sg::swiglu(gate, up);
}
// For bf16 results: with E = e^-|g| = h h, silu(g) is g / (1 + E), and g E / (1 + E) below
// 0. There g takes one h and the up the other, so that neither what is small nor what is
// large leaves 32 bits before the result does (1 + e^-g would be infinite from -89 on, and
// its reciprocal below the normal numbers from -87; here gates below -174 give 0).
__device__ __forceinline__ float swiglu(float gate, float up, uint16_t) {
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(gate) * -0.7213475204444817f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.f)));
  const float a = gate < 0.f ? h : 1.f;
  return gate * a * r * (up * a);
}

// --- Few tokens: a cluster per adapter -----------------------------------------
// Up to kFew tokens in any order, kThreads of them looked at together. Cluster c stands
// for token c: it is at work if the number of earlier ones with the same adapter is a
// multiple of kGroup, and takes those of the next kGroup (this token the first) at
// once. So weights are read once for eight tokens that share them, wherever they stand.
//
// Weights are the 16 rows of m16n8k16, the tokens its 8 columns. A warp takes 32
// outputs at a time, two products: row g + 8 h of product t is output
// 4 g + 2 t + h, so that a lane has four outputs in a row of two tokens. B's
// first rows are on their way before the cluster's sums are there.
//
// kFew: tokens whose neighbours have other adapters are runs of one to the other kernel,
// a round of which takes as long as one of 96. us there / here, 512 tokens on 4096 x
// 6144, rank 32: fp32 one run 28 / 20, six 40 / 23, 48 adapters at random 644 / 37; bf16
// 16 / 17, 23 / 18, 334 / 33. 1024 tokens in six runs: 46 / 43, 26 / 33.
constexpr int kFew = 2 * kThreads, kGroup = 8;
// CTAs of a cluster: eight for up to kWide tokens, or where an adapter has more than
// kLong outputs, else four: 61 tokens on 4096 x 6144, rank 16, 10.9 us with eight and
// 11.4 with four, 128 tokens 14.7 and 13.3, 256 tokens 21 and 18; 61 on 4096 x 28672,
// rank 64, 33 and 60.
constexpr int kWide = 64, kLong = 8192;

// U units of 32 ranks.
template <int U>
struct Few {
  static constexpr int kRow = 32 * U + 4;                     // floats of a token's sums
  static constexpr size_t bytes(int ctas) {
    return sizeof(float) * (kWarps + ctas) * kGroup * kRow;
  }
};

// Eight consecutive bf16 weights of two rows, as the A operands of two k16
// steps; columns of both steps are in the same order as in the B operands.
__device__ __forceinline__ void operands(uint4 lo, uint4 hi, uint32_t (&a)[2][4]) {
  a[0][0] = lo.x; a[0][1] = hi.x; a[0][2] = lo.y; a[0][3] = hi.y;
  a[1][0] = lo.z; a[1][1] = hi.z; a[1][2] = lo.w; a[1][3] = hi.w;
}
__device__ __forceinline__ uint4 load_if(bool in, const uint16_t* p) {
  return in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

template <typename T, int CTAS, int U>
__global__ void __launch_bounds__(kThreads, U <= 2 ? 2 : 1) k_lora_few(const LoraArgs p) {
  using F = Few<U>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kXParts = kF32 ? 3 : 1, kSParts = kF32 ? 3 : 2;
  constexpr int kRow = F::kRow;
  extern __shared__ __align__(16) float smem[];
  float* const sums = smem;                                // [warp][token][kRow]
  float* const exchange = smem + kWarps * kGroup * kRow;   // [cta][token][kRow]
  __shared__ int members[kGroup], before[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = threadIdx.x;
  const int g8 = lane >> 2, c4 = lane & 3;
  const uint32_t cta = cluster_rank();
  const int token = blockIdx.x / CTAS;
  sg::pdl_trigger();
  sg::pdl_wait();
  // Adapter of token i, -1 for none.
  auto adapter = [&](int i) {
    const int id = p.adapter[i];
    return id >= 0 && id < p.adapters ? id : -1;
  };
  const int mine = token / kThreads * kThreads + me;  // this thread's token
  const int id = mine < p.m ? adapter(mine) : -2, d = adapter(token);
  const int earlier = __syncthreads_count(mine < token && id == d);
  if (earlier % kGroup) return;  // the same in all CTAs of the cluster
  cluster_started();
  const unsigned peers = __ballot_sync(0xFFFFFFFFu, mine >= token && id == d);
  if (lane == 0) before[warp] = __popc(peers);
  __syncthreads();
  int at = __popc(peers & ((1u << lane) - 1)), count = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) at += before[w];
    count += before[w];
  }
  if ((peers >> lane & 1) && at < kGroup) members[at] = mine;
  count = min(count, kGroup);
  __syncthreads();

  // This CTA's outputs, in tiles of 32, one in kWarps to each warp.
  const int tiles = (p.n + 31) / 32, share = (tiles + CTAS - 1) / CTAS;
  const int tile1 = min(tiles, (int)(cta + 1) * share);
  int tile = cta * share + warp;
  // Row h of product t for this lane, ranks 32 u + 8 c4 to 32 u + 8 c4 + 7.
  const uint16_t* const b = p.b + (size_t)max(d, 0) * p.n * p.rank + 8 * c4;
  auto load_rows = [&](int tile, uint4 (&w)[U][4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int n = 32 * tile + 4 * g8 + i;
#pragma unroll
      for (int u = 0; u < U; u++)
        w[u][i] = load_if(d >= 0 && tile < tile1 && n < p.n && 32 * u + 8 * c4 < p.rank,
                          b + (size_t)n * p.rank + 32 * u);
    }
  };
  // This lane's two tokens, and its four base entries of each.
  const bool in0 = 2 * c4 < count, in1 = 2 * c4 + 1 < count;
  const size_t token0 = members[in0 ? 2 * c4 : 0], token1 = members[in1 ? 2 * c4 + 1 : 0];
  auto load_base = [&](int tile, float (&v)[2][4]) {
    const int n = 32 * tile + 4 * g8, last = tile < tile1 ? max(0, min(4, p.n - n)) : 0;
    const T* const base = static_cast<const T*>(p.base);
    load<4>(base + token0 * p.ldb + n, v[0], in0 && p.base ? last : 0, p.wide);
    load<4>(base + token1 * p.ldb + n, v[1], in1 && p.base ? last : 0, p.wide);
  };
  uint4 w[U][4];
  float base[2][4];
  load_rows(tile, w);
  load_base(tile, base);

  // A x: this CTA's steps of 32 entries, one in kWarps to each warp. This lane's
  // column is token g8.
  if (d >= 0) {
    const int steps = (p.k + 31) / 32, per = (steps + CTAS - 1) / CTAS;
    const int step1 = min(steps, (int)(cta + 1) * per);
    const uint16_t* const a = p.a + (size_t)d * p.rank * p.k;
    const T* const x = static_cast<const T*>(p.x) + (size_t)members[g8 < count ? g8 : 0] * p.ldx;
    float acc[2 * U][4];
#pragma unroll
    for (int j = 0; j < 2 * U; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    for (int s = cta * per + warp; s < step1; s += kWarps) {
      const int k0 = 32 * s + 8 * c4;
      const bool in = k0 < p.k;
      uint4 y[2 * U][2];
#pragma unroll
      for (int j = 0; j < 2 * U; j++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          y[j][h] = load_if(in && 16 * j + 8 * h < p.rank,
                            a + (size_t)(16 * j + 8 * h + g8) * p.k + k0);
      float v[8];
      load<8>(x + k0, v, in && g8 < count ? 8 : 0, true);
      uint32_t xb[kXParts][4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (kF32)
          parts<3>(v[2 * i], v[2 * i + 1], &xb[0][i], 4);
        else
          xb[0][i] = upper(v[2 * i], v[2 * i + 1]);
      }
#pragma unroll
      for (int j = 0; j < 2 * U; j++) {
        if (16 * j >= p.rank) break;
        uint32_t ya[2][4];
        operands(y[j][0], y[j][1], ya);
        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = kXParts - 1; q >= 0; q--) {
          mma_bf16(z, ya[0], xb[q][0], xb[q][1]);
          mma_bf16(z, ya[1], xb[q][2], xb[q][3]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) acc[j][e] += z[e];
      }
    }
    float* const to = sums + (warp * kGroup + 2 * c4) * kRow + g8;
#pragma unroll
    for (int j = 0; j < 2 * U; j++) {
      if (16 * j >= p.rank) break;
      to[16 * j] = acc[j][0];
      to[16 * j + kRow] = acc[j][1];
      to[16 * j + 8] = acc[j][2];
      to[16 * j + 8 + kRow] = acc[j][3];
    }
  }
  __syncthreads();
  cluster_wait();
  // The warps' sums, to all CTAs; then the CTAs' sums.
  if (d >= 0)
    for (int e = me; e < count * p.rank; e += kThreads) {
      const int at = e / p.rank * kRow + e % p.rank;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; i++) v += sums[i * kGroup * kRow + at];
#pragma unroll
      for (uint32_t c = 0; c < CTAS; c++) store_to(exchange + cta * kGroup * kRow + at, c, v);
    }
  cluster_sync();
  if (d >= 0) {
    const float scale = p.scale ? p.scale[d] : 1.f;
    for (int e = me; e < count * p.rank; e += kThreads) {
      const int at = e / p.rank * kRow + e % p.rank;
      float v = 0.f;
#pragma unroll
      for (int c = 0; c < CTAS; c++) v += exchange[c * kGroup * kRow + at];
      sums[at] = v * scale;
    }
  }
  __syncthreads();
  uint32_t sb[U][kSParts][4];
#pragma unroll
  for (int u = 0; u < U; u++) {
    float v[8];
    load<8>(sums + g8 * kRow + 32 * u + 8 * c4, v,
            d >= 0 && g8 < count && 32 * u + 8 * c4 < p.rank ? 8 : 0, true);
#pragma unroll
    for (int i = 0; i < 4; i++) parts<kSParts>(v[2 * i], v[2 * i + 1], &sb[u][0][i], 4);
  }

  for (; tile < tile1; tile += kWarps) {
    float big[2][4], small[2][4];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) big[t][e] = small[t][e] = 0.f;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        uint32_t wa[2][4];
        operands(w[u][2 * t], w[u][2 * t + 1], wa);
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int q = kSParts - 1; q > 0; q--)
            mma_bf16(small[t], wa[h], sb[u][q][2 * h], sb[u][q][2 * h + 1]);
          mma_bf16(big[t], wa[h], sb[u][0][2 * h], sb[u][0][2 * h + 1]);
        }
      }
    float v[2][4];
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int j = 0; j < 4; j++)  // product j / 2, row j % 2
        v[e][j] = base[e][j] + (big[j / 2][2 * (j % 2) + e] + small[j / 2][2 * (j % 2) + e]);
    load_rows(tile + kWarps, w);
    load_base(tile + kWarps, base);
    const int n = 32 * tile + 4 * g8, last = tile < tile1 ? max(0, min(4, p.n - n)) : 0;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (!(e ? in1 : in0) || !last) continue;
      T* const row = static_cast<T*>(p.out) + (e ? token1 : token0) * p.ldo;
      if (p.epi == STRASGPT_EPI_SWIGLU) {
        const float y[2] = {swiglu(v[e][0], v[e][1], T()), swiglu(v[e][2], v[e][3], T())};
        store<2>(row + n / 2, y, last / 2, p.wide);
      } else {
        if (p.epi == STRASGPT_EPI_ADD) {
          float old[4];
          load<4>(row + n, old, last, p.wide);
#pragma unroll
          for (int j = 0; j < 4; j++) v[e][j] += old[j];
        }
        store<4>(row + n, v[e], last, p.wide);
      }
    }
  }
}

template <typename T, int CTAS, int U>
cudaError_t launch_few(const LoraArgs& p, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  constexpr size_t bytes = Few<U>::bytes(CTAS);
  const cudaError_t e = sg::allow_smem(k_lora_few<T, CTAS, U>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  return sg::try_launch(k_lora_few<T, CTAS, U>, dim3((unsigned)p.m * CTAS), dim3(kThreads), bytes,
                        CTAS, s, p);
}

template <typename T, int CTAS>
cudaError_t launch_few_rank(const LoraArgs& p, int dev, cudaStream_t s) {
  if (p.rank <= 32) return launch_few<T, CTAS, 1>(p, dev, s);
  if (p.rank <= 64) return launch_few<T, CTAS, 2>(p, dev, s);
  return launch_few<T, CTAS, 4>(p, dev, s);
}

// --- Many tokens -----------------------------------------------------------------
// A cluster has tiles of consecutive tokens, and takes a tile's runs of one
// adapter one after the other. The tokens are the 128 rows of tcgen05 products, of
// A x and then of B (A x). There are two sides, for even and odd stages of both
// products, each with a ring of its own: a warp that brings in what the others need
// by TMA, one that issues the matrix instructions, and a warpgroup that works on
// rows. (Two, because a stage costs a warp that asks or issues some hundred cycles of
// waits, whatever its size; apart, because a wait on a barrier's parity needs who
// waits for all of its phases.)
//
// A x: a stage has 128 bytes of the tokens' rows, and A's entries beside them. bf16
// rows are operands as they are; fp32 rows become bf16 parts in shared memory.
//
// B (A x): a stage has 128 bytes of the tokens' base rows, and B's for as many
// outputs. A x lies in shared memory, as bf16 parts. The sums go to one of kSlots
// places in tensor memory. A thread has a token, adds its sums to the base row in the
// stage, where the results take their place, and each warp sends its 32 rows off by TMA.
constexpr int kManyThreads = kThreads + 128;
constexpr int kSlots = 2, kMaxStages = 4;  // of a side
constexpr int kChunks = 256;  // of 32 tokens that are looked over at a time
constexpr unsigned long long kTimeoutNs = 2000000000ULL;

// P panels of 64 ranks.
template <typename T, int P>
struct Many {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kXParts = kF32 ? 3 : 1, kParts = kF32 ? 3 : 2;  // of x, of A x
  static constexpr int kCols = 128 / (int)sizeof(T);   // of a stage: x's entries, or outputs
  static constexpr int kSide = 64 * kCols * 2;         // bytes: A's or B's entries of 64 ranks
  static constexpr int kXBuffers = 2;                  // fp32 x: a warpgroup's stage as parts
  static constexpr int kRow = 64 * P + 4;              // floats of a token in the exchange
  // Shared memory: A x as an operand (parts of x in its place before), then the
  // ring (the cluster's exchange in its place between the products).
  static constexpr int kMemory = (P == 1 ? 108 : 220) * 1024, kBytes = kMemory + 1024;
  // Tensor memory: the slots; A x's sums (fp32: those of the first part, and of
  // the others), of each issuing warp, in their place.
  static constexpr int kSums = (kF32 ? 2 : 1) * 64 * P;
  static constexpr int kColumns = 2 * (kSums > kSlots * kCols ? kSums : kSlots * kCols);
  // fp32 sums of bf16 products, 128 rows; columns to be added.
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);
};

// What tiles of `tokens` tokens (a multiple of 32) make of it: bytes.
struct Layout {
  int panel;    // a tile's 128-byte rows: of x, of base, of 64 ranks of A x
  int operand, stage, stages;  // stages: of a side
};
template <typename T, int P>
Layout layout_of(int tokens, bool both) {
  using M = Many<T, P>;
  Layout l;
  l.panel = tokens * 128;
  l.operand = M::kParts * P * l.panel;
  l.stage = l.panel * (both ? 2 : 1) + P * M::kSide;
  // Operands have 128 rows, whatever the tile has: what lies behind is read too
  // (and comes to nothing), so that behind the last stage there is room. (There is one
  // stage at least, for tiles of up to 96 tokens.)
  const int room = M::kMemory - l.operand - std::max(0, kMaxTokens * 128 - l.stage);
  l.stages = std::min(kMaxStages, room / l.stage / 2);
  return l;
}

struct ManyMaps {
  CUtensorMap x, a, b, base, out;
};

__device__ __forceinline__ uint32_t saddr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait of a whole warp, which stays together; false once any wait of the
// CTA has run out (`always`: waits all the same, for what was asked for).
__device__ __forceinline__ bool warp_wait(uint32_t bar, unsigned parity, volatile int* failed,
                                          bool always = false) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const unsigned long long t0 = now_ns();
    while (!(ok = mbar_try_wait(bar, parity))) {
      if (*failed && !always) break;
      if (now_ns() - t0 > kTimeoutNs) {
        *failed = 1;
        break;
      }
    }
  }
  return __all_sync(0xFFFFFFFFu, ok);
}
__device__ __forceinline__ uint32_t elect() {
  uint32_t one;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(one));
  return one;
}
__device__ __forceinline__ void mbar_arrive7(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 7;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive2(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 2;" ::"r"(bar) : "memory");
}
// Boxes of matrices (x is a multiple of 64 bytes); zeros outside.
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                       uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                       uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// The other way, and until the boxes sent have been read (`read`) or written.
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}
template <int LEFT>
__device__ __forceinline__ void tma_store_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void tma_store_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// K-major operand of 128-byte rows with 128-byte swizzle, 8-row atoms of 1024
// bytes; of 64-byte rows with 64-byte swizzle, atoms of 512.
__device__ __forceinline__ uint64_t swizzled(uint32_t addr, int row_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 |
         (uint64_t)(8 * row_bytes >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)(row_bytes == 128 ? 2 : 4) << 61;
}
// The matrix instructions are issued under a predicate and not in a branch, so
// that their operands can stay in uniform registers.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add, uint32_t issue) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t issue) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
          bar),
      "r"(issue)
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Orders this thread's accesses to shared memory with the tensor cores' and
// TMA's.
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void fence_async_cluster() {
  asm volatile("fence.proxy.async.shared::cluster;" ::: "memory");
}
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// Entry e of a 128-byte row that lies in a swizzled tile.
template <typename T>
__device__ __forceinline__ T* entry(uint8_t* row, int r, int e) {
  constexpr int kV = 16 / sizeof(T);
  return reinterpret_cast<T*>(row + (((e / kV) ^ (r & 7)) << 4)) + e % kV;
}

// A warp reads `outs` entries each of `mine` rows, ld apart, into a swizzled tile. Several
// rows are on their way at once (636 fp32 tokens on 776 x 2803, rank 8, 40 us one after
// the other, now 33), and apart from the rows that TMA brings, which need its registers.
template <typename T>
__device__ __noinline__ void read_rows(uint8_t* rows, const T* from, long long ld, int mine,
                                          int outs) {
  constexpr int kOf = 128 / (int)sizeof(T) / 32, kAtOnce = 16 / kOf;  // entries a lane; rows
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int j0 = 0; j0 < mine; j0 += kAtOnce) {
    T v[kAtOnce][kOf];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)
#pragma unroll
      for (int e = 0; e < kOf; e++)
        v[j][e] = j0 + j < mine && lane + 32 * e < outs ? from[(j0 + j) * ld + lane + 32 * e]
                                                        : T(0);
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)
#pragma unroll
      for (int e = 0; e < kOf; e++)
        if (j0 + j < mine) *entry<T>(rows + (j0 + j) * 128, j0 + j, lane + 32 * e) = v[j][e];
  }
}

// Adds 32 entries of a row that lies swizzled in a tile (its first or second 64
// bytes: bf16; all of it: fp32).
template <typename T>
__device__ __forceinline__ void add_row(const uint8_t* row, int r, int half, float (&v)[32]) {
  constexpr int kV = 16 / (int)sizeof(T);
#pragma unroll
  for (int c = 0; c < 32 / kV; c++) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + (((half * 4 + c) ^ (r & 7)) << 4));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) {
        v[4 * c + i] += __uint_as_float(u[i]);
      } else {
        v[8 * c + 2 * i] += sg::bf16_lo(u[i]);
        v[8 * c + 2 * i + 1] += sg::bf16_hi(u[i]);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 packed(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  else
    return make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]),
                      bf16x2(v[6], v[7]));
}

// Sixteen gates and ups in turn -> silu(gate) up, packed. All lanes of a warp call it.
__device__ __forceinline__ void swiglu16(const float (&v)[32], uint4 (&y)[4], float t) {
#pragma unroll
  for (int c = 0; c < 4; c++) {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = swiglu(v[8 * c + 2 * j], v[8 * c + 2 * j + 1], t);
    y[c] = packed<float>(x);
  }
}
// For bf16 results one reciprocal serves two, 1/a = b / (a b): what bounds this is the
// unit of exp and reciprocal. That is good while a b is below 2^120, two gates of -41 or
// one of -83; where one of the warp's pairs is beyond, or has a NaN, each result is
// computed by itself. It is looked for once the results are there, so that nothing waits
// for the vote (before the exponentials it cost 4001 tokens on 4096 x 28672 8 us).
__device__ __forceinline__ void swiglu16(const float (&v)[32], uint4 (&y)[2], uint16_t t) {
  float least = 1.f;  // of the reciprocals
#pragma unroll
  for (int c = 0; c < 2; c++) {
    float x[8], r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float* const p = v + 16 * c + 4 * j;
      float e0, e1;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(p[0] * -1.4426950408889634f));
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(p[2] * -1.4426950408889634f));
      e0 += 1.f;
      e1 += 1.f;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r[j]) : "f"(e0 * e1));
      x[2 * j] = p[0] * (r[j] * e1) * p[1];
      x[2 * j + 1] = p[2] * (r[j] * e0) * p[3];
    }
    asm("min.NaN.f32 %0, %0, %1, %2;" : "+f"(least) : "f"(r[0]), "f"(r[1]));
    asm("min.NaN.f32 %0, %0, %1, %2;" : "+f"(least) : "f"(r[2]), "f"(r[3]));
    y[c] = packed<uint16_t>(x);
  }
  if (!__all_sync(0xFFFFFFFFu, least >= 0x1p-120f)) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = swiglu(v[16 * c + 2 * j], v[16 * c + 2 * j + 1], t);
      y[c] = packed<uint16_t>(x);
    }
    __syncwarp();
  }
}

// Sixteen entries of a row of a stage of fp32 x -> the same place in three parts'
// rows of 64 bytes, 64-byte swizzle.
__device__ __forceinline__ void split_row(const uint8_t* row, int r, int half, uint8_t* to,
                                          int part) {
  uint32_t w[3][8];
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const float4 v = *reinterpret_cast<const float4*>(row + (((half * 4 + c) ^ (r & 7)) << 4));
    parts<3>(v.x, v.y, &w[0][2 * c], 8);
    parts<3>(v.z, v.w, &w[0][2 * c + 1], 8);
  }
#pragma unroll
  for (int q = 0; q < 3; q++)
#pragma unroll
    for (int c = 0; c < 2; c++)
      *reinterpret_cast<uint4*>(to + q * part + r * 64 +
                                (((half * 2 + c) ^ ((r >> 1) & 3)) << 4)) =
          make_uint4(w[q][4 * c], w[q][4 * c + 1], w[q][4 * c + 2], w[q][4 * c + 3]);
}

// The value of lane 0, known to be the same in all lanes.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

// A warp's place among the fills of its side's ring, or its slots.
struct Place {
  int at = 0;
  unsigned phase = 0;  // parity of the present one
  __device__ __forceinline__ void next(int places) {
    if (++at == places) {
      at = 0;
      phase ^= 1;
    }
  }
};

// Calls f(first token, tokens, adapter or -1) for each of this cluster's items: an
// item is a run of one adapter in a tile of p.tokens tokens, and each cluster has
// every clusters-th. All threads of the cluster's CTAs take part, and have arrived at
// the cluster's barrier.
template <typename F>
__device__ __forceinline__ void each_item(const LoraArgs& p, unsigned* starts, int* before, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, clusters = gridDim.x / kCluster;
  const uint32_t cta = cluster_rank();
  int turn = blockIdx.x / kCluster;  // items until this cluster's next
  auto adapter = [&](int t) {
    const int id = p.adapter[t];
    return id >= 0 && id < p.adapters ? id : -1;
  };
#pragma unroll 1
  for (int w0 = 0; w0 < p.m;) {
    const int wn = min(32 * kChunks, p.m - w0), chunks = (wn + 31) / 32;
    if (w0) cluster_arrive();
    cluster_wait();  // all are there, and done with the last ones
    // Each CTA looks over every kCluster-th chunk for all of them.
#pragma unroll 1
    for (int c = warp * kCluster + cta; c < chunks; c += kManyThreads / 32 * kCluster) {
      const int i = 32 * c + lane;
      const bool in = i < wn;
      const int id = in ? adapter(w0 + i) : -1, before = in && i ? adapter(w0 + i - 1) : -1;
      const unsigned mask = __ballot_sync(0xFFFFFFFFu, in && (i % p.tokens == 0 || id != before));
      if (lane < kCluster)
        store_to(reinterpret_cast<float*>(starts + c), lane, __uint_as_float(mask));
    }
    cluster_sync();
    if (warp == 0) {
      int sum = 0;
      for (int c0 = 0; c0 < chunks; c0 += 32) {
        const int mine = c0 + lane < chunks ? __popc(starts[c0 + lane]) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
          if (lane >= o) upto += x;
        }
        if (c0 + lane < chunks) before[c0 + lane] = sum + upto - mine;
        sum += __shfl_sync(0xFFFFFFFFu, upto, 31);
      }
      if (lane == 0) before[chunks] = sum;
    }
    __syncthreads();
    const int items = before[chunks];
#pragma unroll 1
    for (; turn < items; turn += clusters) {
      // Item `turn`: its chunk, its bit there, and the next item's.
      int c = 0;
      for (int step = kChunks / 2; step > 0; step /= 2)
        if (c + step < chunks && before[c + step] <= turn) c += step;
      unsigned bits = starts[c];
      for (int skip = turn - before[c]; skip > 0; skip--) bits &= bits - 1;
      const int r0 = 32 * c + __ffs(bits) - 1;
      bits &= bits - 1;
      while (!bits && ++c < chunks) bits = starts[c];
      const int count = (bits ? 32 * c + __ffs(bits) - 1 : wn) - r0;
      f(w0 + r0, count, adapter(w0 + r0));
    }
    turn -= items;
    w0 += wn;
  }
}

// What bounds it: in the second product, memory and its latency (1.3 us from a
// stage's request to its arrival, two stages a side of 96 tokens: 5.7 TB/s while all
// SMs are at it); over the whole, that items come in rounds of the 33 or so clusters
// that the GPU holds (46 items of 4001 tokens in five runs make two rounds) and that an
// item takes 20 us before its first output (finding it 4, A x 6, the exchange 6). Tiles
// of 128 tokens have room for one stage a side: 4001 tokens in five runs 221 us, now 144.
template <typename T, int P>
__global__ void __launch_bounds__(kManyThreads, P == 1 ? 2 : 1)
    k_lora_many(const LoraArgs p, const Layout l, const __grid_constant__ ManyMaps maps) {
  using M = Many<T, P>;
  constexpr bool kF32 = M::kF32;
  constexpr int kParts = M::kParts, kCols = M::kCols, kHalves = kCols / 32, kRow = M::kRow;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t filled_[2][kMaxStages], frees_[2][kMaxStages],
      full_[2][kSlots], empty_[2][kSlots], x_full[M::kXBuffers], x_empty[M::kXBuffers],
      sums_full, done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ unsigned starts[kChunks];
  __shared__ int before[kChunks + 1];
  // The same in all lanes, and known to be: what TMA and the matrix instructions
  // are given stays in uniform registers.
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool worker = warp < kWarps, loader = !worker && warp < kWarps + 2;
  const int side_of = worker ? warp >> 2 : warp & 1;  // its stages: even, odd ones
  const uint32_t cta = cluster_rank(), s_at = (saddr(raw) + 1023u) & ~1023u;
  cluster_started();
  uint8_t* const operand = raw + (s_at - saddr(raw));
  const uint32_t ring_at = s_at + l.operand + side_of * l.stages * l.stage;
  uint8_t* const ring = operand + l.operand + side_of * l.stages * l.stage;
  uint64_t *const filled = filled_[side_of], *const free_ = frees_[side_of],
                  *const full = full_[side_of], *const empty = empty_[side_of];
  sg::pdl_trigger();
  sg::pdl_wait();
  if (threadIdx.x == 0) {
    for (int side = 0; side < 2; side++) {
      for (int s = 0; s < kMaxStages; s++) {
        mbar_init(saddr(&filled_[side][s]), 1);
        mbar_init(saddr(&frees_[side][s]), 8);
      }
      for (int s = 0; s < kSlots; s++) {
        mbar_init(saddr(&full_[side][s]), 1);
        mbar_init(saddr(&empty_[side][s]), 4);
      }
    }
    for (int b = 0; b < M::kXBuffers; b++) {
      mbar_init(saddr(&x_full[b]), 4);
      mbar_init(saddr(&x_empty[b]), 1);
    }
    mbar_init(saddr(&sums_full), 2);
    mbar_init(saddr(&done), 2);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kWarps + 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     saddr(&tmem_slot)),
                 "r"(M::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);
  // Old values that are added: base's, and out's.
  const bool gated = p.epi == STRASGPT_EPI_SWIGLU, old = p.epi == STRASGPT_EPI_ADD;
  const bool both = old && p.base, has = old || p.base;
  const int stages = l.stages, side = l.panel;  // of a stage: where A's or B's entries lie
  const int second = l.panel + P * M::kSide;    // and, if both are added, out's rows
  const int x_part = p.tokens * kCols * 2;      // bytes of a part of a stage's x
  Place stage;
  auto wait_filled = [&] { return warp_wait(saddr(&filled[stage.at]), stage.phase, &failed); };
  // This CTA's share of the entries and of the outputs, in stages.
  const int k_stages = (p.k + kCols - 1) / kCols, k_share = (k_stages + kCluster - 1) / kCluster;
  const int k0 = cta * k_share, k_mine = max(0, min(k_stages, k0 + k_share) - k0);
  const int n_units = (p.n + kCols - 1) / kCols, n_share = (n_units + kCluster - 1) / kCluster;
  const int n0 = cta * n_share, n_mine = max(0, min(n_units, n0 + n_share) - n0);
  const int steps = (p.rank + 15) / 16;

  // Each role goes through the same items and barriers. P 1, two CTAs to an SM: 384
  // threads of 80 registers, which 256 of 96 and 128 of 48 are.
  if (!worker) {
    if constexpr (P == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    const uint32_t one = elect();
    // The exchange of A x is the workers'.
    auto exchanged = [&] {
      cluster_sync();
      cluster_sync();
      fence_async();
      __syncthreads();
      fence_after();
    };
    if (loader) {
      bool dead = false;  // nothing is asked for after a wait that ran out
      int issued = 0;
      // (The first wait on a barrier, for the phase before its first, ends at once.)
      auto ask = [&](auto boxes) {
        dead = dead || !warp_wait(saddr(&free_[stage.at]), stage.phase ^ 1, &failed);
        if (dead) return;
        issued++;
        if (one) boxes(ring_at + stage.at * l.stage, saddr(&filled[stage.at]));
        __syncwarp();
        stage.next(stages);
      };
      each_item(p, starts, before, [&](int token0, int count, int d) {
        const int boxes = (count + 31) / 32;
        if (d >= 0) {
#pragma unroll 1
          for (int i = side_of; i < k_mine; i += 2) {
            ask([&](uint32_t at, uint32_t bar) {
              mbar_expect_tx(bar, boxes * 4096 + P * M::kSide);
              for (int b = 0; b < boxes; b++)
                tma_2d(at + b * 4096, &maps.x, (k0 + i) * kCols, token0 + 32 * b, bar);
#pragma unroll
              for (int j = 0; j < P; j++)
                tma_3d(at + side + j * M::kSide, &maps.a, (k0 + i) * kCols, 64 * j, d, bar);
            });
          }
          exchanged();
        }
        const uint32_t bytes = (d >= 0 ? P * M::kSide : 0) +
                               (p.base_tma ? boxes * 4096 * (both ? 2 : 1) : 0);
#pragma unroll 1
        for (int i = side_of; i < n_mine; i += 2) {
          ask([&](uint32_t at, uint32_t bar) {
            const int n = (n0 + i) * kCols;
            mbar_expect_tx(bar, bytes);
            if (d >= 0) {
#pragma unroll
              for (int j = 0; j < P; j++)
                tma_3d(at + side + j * M::kSide, &maps.b, 64 * j, n, d, bar);
            }
            if (p.base_tma)
              for (int b = 0; b < boxes; b++) {
                tma_2d(at + b * 4096, p.base ? &maps.base : &maps.out, n, token0 + 32 * b, bar);
                if (both) tma_2d(at + second + b * 4096, &maps.out, n, token0 + 32 * b, bar);
              }
          });
        }
      });
      // Nothing asked for outlives the ring: each stage's last fill, the
      // (issued - 1 - s) / stages-th, has landed.
      for (int s = 0; s < min(stages, issued); s++)
        warp_wait(saddr(&filled[s]), ((issued - 1 - s) / stages) & 1, &failed, true);
    } else {
      Place slot;
      unsigned x_phase = 0;
      each_item(p, starts, before, [&](int, int, int d) {
        if (d < 0) {
          for (int i = side_of; i < n_mine; i += 2) stage.next(stages);
          return;
        }
        // The workers are past the last slots: the sums may take their place.
        asm volatile("bar.sync 1, 320;" ::: "memory");
        {
          const uint32_t idesc = M::kIdesc | (uint32_t)(2 * steps) << 17;
          const uint32_t to = uniform(tmem + side_of * M::kSums);
          const uint64_t x0 = swizzled(uniform(s_at + side_of * M::kXParts * x_part), kCols * 2);
#pragma unroll 1
          for (int i = side_of; i < k_mine; i += 2, stage.next(stages)) {
            bool ok = wait_filled();
            if (kF32) ok = ok && warp_wait(saddr(&x_full[side_of]), x_phase, &failed);
            const uint32_t at = uniform(ring_at + stage.at * l.stage);
            if (ok) {
              fence_after();
              const uint64_t b0 = swizzled(at + side, kCols * 2);
              if constexpr (kF32) {
#pragma unroll
                for (int q = 2; q >= 0; q--)
#pragma unroll
                  for (int k = 0; k < 2; k++)
                    mma_ss(to + (q ? 64 * P : 0), x0 + ((q * x_part + k * 32) >> 4), b0 + 2 * k,
                           idesc, i > 1 || k > 0 || q == 1, one);
              } else {
                const uint64_t a0 = swizzled(at, 128);
#pragma unroll
                for (int k = 0; k < 4; k++)
                  mma_ss(to, a0 + 2 * k, b0 + 2 * k, idesc, i > 1 || k > 0, one);
              }
            }
            // The stage is free once these have been executed: one of eight arrivals.
            // (The workers, who read it before, need not arrive.)
            if (one) mbar_arrive7(saddr(&free_[stage.at]));
            mma_commit(saddr(&free_[stage.at]), one);
            if (kF32) {
              mma_commit(saddr(&x_empty[side_of]), one);
              x_phase ^= 1;
            }
          }
          mma_commit(saddr(&sums_full), one);
        }
        exchanged();
        const uint32_t idesc = M::kIdesc | (uint32_t)(kCols / 8) << 17;
        const uint64_t a0 = swizzled(uniform(s_at), 128);
#pragma unroll 1
        for (int i = side_of; i < n_mine; i += 2, stage.next(stages), slot.next(kSlots)) {
          const bool ok =
              wait_filled() && warp_wait(saddr(&empty[slot.at]), slot.phase ^ 1, &failed);
          const uint64_t b0 = swizzled(uniform(ring_at + stage.at * l.stage + side), 128);
          const uint32_t to = uniform(tmem + (side_of * kSlots + slot.at) * kCols);
          if (ok) {
            fence_after();
            // (Unrolled: with offsets to be computed an instruction takes 140 cycles, not
            // 30.)
#pragma unroll
            for (int q = kParts - 1; q >= 0; q--)
#pragma unroll
              for (int j = 0; j < P; j++) {
                const uint64_t aq = a0 + (uint32_t)((q * P + j) * l.panel >> 4);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  if (4 * j + k >= steps) break;
                  mma_ss(to, aq + 2 * k, b0 + ((j * M::kSide + k * 32) >> 4), idesc,
                         q < kParts - 1 || j + k > 0, one);
                }
              }
          }
          mma_commit(saddr(&full[slot.at]), one);
        }
      });
      // Nothing issued outlives the tensor memory.
      mma_commit(saddr(&done), one);
      warp_wait(saddr(&done), 0, &failed, true);
    }
  } else {
    if constexpr (P == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    const int quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
    Place slot;
    unsigned x_phase = 0, sums_phase = 0;
    each_item(p, starts, before, [&](int token0, int count, int d) {
      if (d >= 0) {
        asm volatile("bar.sync 1, 320;" ::: "memory");
#pragma unroll 1
        for (int i = side_of; i < k_mine; i += 2, stage.next(stages)) {
          if (!kF32) continue;
          const bool ok =
              wait_filled() && warp_wait(saddr(&x_empty[side_of]), x_phase ^ 1, &failed);
          x_phase ^= 1;
          if constexpr (kF32) {
            if (ok && r < (count + 31) / 32 * 32) {
              const uint8_t* const row = ring + stage.at * l.stage + r * 128;
              uint8_t* const to = operand + side_of * M::kXParts * x_part;
              split_row(row, r, 0, to, x_part);
              split_row(row, r, 1, to, x_part);
            }
          }
          fence_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(saddr(&x_full[side_of]));
        }
        // The sums of all of this CTA's entries; the ring and the operand's place are
        // read.
        warp_wait(saddr(&sums_full), sums_phase, &failed);
        sums_phase ^= 1;
        fence_after();
        // They go to shared memory; a thread has a token's first or second 32 P ranks.
        float* const sums = reinterpret_cast<float*>(operand + l.operand);
        {
          const int c0 = side_of * 32 * P;
#pragma unroll
          for (int c = 0; c < 32 * P; c += 32) {
            if (c0 + c >= p.rank) break;
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.f;
#pragma unroll 1
            for (int set = 0; set < min(2, k_mine); set++) {
#pragma unroll
              for (int part = kF32 ? 1 : 0; part >= 0; part--) {  // small ones first
                float z[32];
                tmem_ld32(lanes + set * M::kSums + part * 64 * P + c0 + c, z);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] += z[j];
              }
            }
            if (r < count) {
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<float4*>(sums + r * kRow + c0 + c + j) =
                    make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
          }
          fence_before();
        }
        cluster_sync();
        // CTA c adds up the cluster's sums of tokens c, c + 8, ..., read from all (in
        // whole rows: they come in packets of 128 bytes), and sends the result to all, as
        // parts: eight ranks a thread, zeros behind the last.
        {
          const float scale = p.scale ? p.scale[d] : 1.f;
          const int c = threadIdx.x % (8 * P);
          for (int row = (int)(threadIdx.x / (8 * P)) * kCluster + cta; row < count;
               row += kThreads / (8 * P) * kCluster) {
            if (c >= 2 * steps) break;
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (8 * c < p.rank) {
              float4 x[2 * kCluster];
#pragma unroll
              for (uint32_t from = 0; from < kCluster; from++) {
                x[2 * from] = load4_from(sums + row * kRow + 8 * c, from);
                x[2 * from + 1] = load4_from(sums + row * kRow + 8 * c + 4, from);
              }
#pragma unroll
              for (int from = 0; from < kCluster; from++) {
                const float4 y = x[2 * from], z = x[2 * from + 1];
                v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
                v[4] += z.x; v[5] += z.y; v[6] += z.z; v[7] += z.w;
              }
            }
            uint32_t w[kParts][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
              parts<kParts>(v[2 * j] * scale, v[2 * j + 1] * scale, &w[0][j], 4);
            uint8_t* const to = operand + (c >> 3) * l.panel + row * 128 + (((c ^ row) & 7) << 4);
#pragma unroll
            for (int q = 0; q < kParts; q++)
#pragma unroll
              for (uint32_t cta_to = 0; cta_to < kCluster; cta_to++)
                store4_to(reinterpret_cast<float*>(to + q * P * l.panel), cta_to,
                          make_float4(__uint_as_float(w[q][0]), __uint_as_float(w[q][1]),
                                      __uint_as_float(w[q][2]), __uint_as_float(w[q][3])));
          }
          fence_async_cluster();
        }
        cluster_sync();
        fence_async();
        __syncthreads();
        fence_after();
      }

      const bool late = stages >= 3;
      const int mine = max(0, min(32, count - 32 * quarter));  // tokens of this warp
#pragma unroll 1
      for (int i = side_of; i < n_mine; i += 2, stage.next(stages)) {
        bool ok = wait_filled();
        const int n = (n0 + i) * kCols, outs = min(kCols, p.n - n);
        uint8_t* const rows = ring + stage.at * l.stage + 32 * quarter * 128;  // the warp's
        uint8_t* const row = rows + lane * 128;
        if (mine && has && !p.base_tma) {
          // Rows that TMA cannot read.
          const T* const b = static_cast<const T*>(p.base ? p.base : p.out);
          const long long ld = p.base ? p.ldb : p.ldo;
          const size_t t = (size_t)token0 + 32 * quarter;
          read_rows(rows, b + t * ld + n, ld, mine, outs);
          if (both)
            read_rows(rows + second, static_cast<const T*>(p.out) + t * p.ldo + n, p.ldo, mine,
                      outs);
          __syncwarp();
        }
        if (d >= 0) {
          ok = warp_wait(saddr(&full[slot.at]), slot.phase, &failed) && ok;
          fence_after();
        }
        if (mine) {
          constexpr int kV = 16 / (int)sizeof(T);
          uint4 y[kHalves][16 / kV];  // of SwiGLU
#pragma unroll
          for (int h = 0; h < kHalves; h++) {
            float v[32];
            if (d >= 0) {
              tmem_ld32(lanes + (side_of * kSlots + slot.at) * kCols + 32 * h, v);
            } else {
#pragma unroll
              for (int j = 0; j < 32; j++) v[j] = 0.f;
            }
            if (has) add_row<T>(row, r, h, v);
            if (both) add_row<T>(row + second, r, h, v);
            if (gated) {
              swiglu16(v, y[h], T());
            } else {
#pragma unroll
              for (int c = 0; c < 32 / kV; c++)
                *reinterpret_cast<uint4*>(row + (((h * 4 + c) ^ (r & 7)) << 4)) =
                    packed<T>(v + kV * c);
            }
          }
          if (gated) {
            // Half as much, in rows of 64 bytes with 64-byte swizzle, where others' base
            // rows were.
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; c++)
              *reinterpret_cast<uint4*>(rows + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
                  y[c / (16 / kV)][c % (16 / kV)];
          }
          // A wait that ran out leaves NaN: no result passes for a complete one.
          if (!ok || failed) {
            __syncwarp();
            for (int c = 0; c < 8; c++)
              *reinterpret_cast<uint4*>(row + 16 * c) = make_uint4(~0u, ~0u, ~0u, ~0u);
          }
          const int x = gated ? n / 2 : n, last = gated ? outs / 2 : outs;
          // (TMA stores whole 16 bytes: where the row ends within them, zeros would take
          // the place of what lies behind it.)
          if (mine == 32 && p.out_tma && last * sizeof(T) % 16 == 0) {
            fence_async();
            __syncwarp();
            if (lane == 0)
              tma_store(&maps.out, x, token0 + 32 * quarter,
                        ring_at + stage.at * l.stage + 32 * quarter * 128);
          } else {
            __syncwarp();
#pragma unroll 4
            for (int j = 0; j < mine; j++) {
              T* const to =
                  static_cast<T*>(p.out) + ((size_t)token0 + 32 * quarter + j) * p.ldo + x;
#pragma unroll
              for (int e = lane; e < kCols; e += 32)
                if (e < last)
                  to[e] = gated ? reinterpret_cast<const T*>(
                                      rows + j * 64 + (((e / kV) ^ ((j >> 1) & 3)) << 4))[e % kV]
                                : *entry<T>(rows + j * 128, j, e);
            }
            fence_async();
          }
        }
        if (d >= 0) fence_before();
        __syncwarp();
        if (lane == 0) {
          if (d >= 0) mbar_arrive(saddr(&empty[slot.at]));
          // The stage is free once its rows are sent. With stages to spare that is
          // waited for a unit later.
          if (late) {
            tma_store_read<1>();
            if (i >= 2)
              mbar_arrive2(saddr(&free_[stage.at ? stage.at - 1 : stages - 1]));
            if (i + 2 >= n_mine) {
              tma_store_read<0>();
              mbar_arrive2(saddr(&free_[stage.at]));
            }
          } else {
            tma_store_read<0>();
            mbar_arrive2(saddr(&free_[stage.at]));
          }
        }
        if (d >= 0) slot.next(kSlots);
      }
    });
    if (lane == 0) tma_store_done();
  }
  __syncthreads();
  if (warp == kWarps + 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(M::kColumns)
                 : "memory");
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::atomic<void*> known;
  void* fn = known.load(std::memory_order_relaxed);
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    known.store(fn, std::memory_order_relaxed);
  }
  return (PFN_cuTensorMapEncodeTiled_v12000)fn;
}

// Map of a row-major matrix (or `deep` of them, `step` entries apart): boxes of
// `cols` entries of `rows` rows.
bool encode_map(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, bool f32,
                const void* base, long long width, long long height, long long ld, int deep,
                int cols, int rows, CUtensorMapSwizzle swizzle) {
  const size_t size = f32 ? 4 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)height, (cuuint64_t)deep};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * size, (cuuint64_t)height * ld * size};
  const cuuint32_t box[3] = {(cuuint32_t)cols, (cuuint32_t)rows, 1}, step[3] = {1, 1, 1};
  return encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                deep ? 3 : 2, const_cast<void*>(base), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters that the GPU holds at once, as far as their SMs go.
int clusters_of(int rank, int sms) { return std::max(1, (rank <= 64 ? 2 : 1) * sms / kCluster); }

template <typename T, int P>
cudaError_t launch_many(const LoraArgs& p, int dev, int sms, cudaStream_t s) {
  const bool both = p.base && p.epi == STRASGPT_EPI_ADD;
  static std::atomic<size_t> allowed[sg::kDevices];
  using M = Many<T, P>;
  const cudaError_t e = sg::allow_smem(k_lora_many<T, P>, M::kBytes, dev, allowed);
  if (e != cudaSuccess) return e;
  const auto encode = encode_fn();
  if (!encode) return cudaErrorNotSupported;
  ManyMaps maps = {};
  const auto sw128 = CU_TENSOR_MAP_SWIZZLE_128B;
  const bool gated = p.epi == STRASGPT_EPI_SWIGLU;
  constexpr int kCols = M::kCols;
  if (!encode_map(encode, &maps.x, M::kF32, p.x, p.k, p.m, p.ldx, 0, kCols, 32, sw128) ||
      !encode_map(encode, &maps.a, false, p.a, p.k, p.rank, p.k, p.adapters, kCols, 64,
                  M::kF32 ? CU_TENSOR_MAP_SWIZZLE_64B : sw128) ||
      !encode_map(encode, &maps.b, false, p.b, p.rank, p.n, p.rank, p.adapters, 64, kCols, sw128) ||
      (p.base && p.base_tma &&
       !encode_map(encode, &maps.base, M::kF32, p.base, p.n, p.m, p.ldb, 0, kCols, 32, sw128)) ||
      (p.out_tma &&
       !(gated ? encode_map(encode, &maps.out, M::kF32, p.out, p.n / 2, p.m, p.ldo, 0, kCols / 2,
                            32, CU_TENSOR_MAP_SWIZZLE_64B)
               : encode_map(encode, &maps.out, M::kF32, p.out, p.n, p.m, p.ldo, 0, kCols, 32,
                            sw128))))
    return cudaErrorInvalidValue;
  const Layout l = layout_of<T, P>(p.tokens, both);
  return sg::try_launch(k_lora_many<T, P>, dim3((unsigned)clusters_of(p.rank, sms) * kCluster),
                        dim3(kManyThreads), M::kBytes, kCluster, s, p, l, maps);
}

template <typename T>
cudaError_t launch_type(const LoraArgs& p, int dev, int sms, cudaStream_t s) {
  if (p.m <= kFew)
    return p.m <= kWide || p.n > kLong ? launch_few_rank<T, 8>(p, dev, s)
                                       : launch_few_rank<T, 4>(p, dev, s);
  return p.rank <= 64 ? launch_many<T, 1>(p, dev, sms, s) : launch_many<T, 2>(p, dev, sms, s);
}

// Tokens of a tile: as few as give each cluster one item at most, if every adapter
// has one run.
int tokens_of(int m, int rank, int adapters, int sms) {
  const int room = std::max(1, clusters_of(rank, sms) - std::min(adapters, 8));
  int t = 32;
  while (t < 96 && m > (long long)t * room) t += 32;
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
  const size_t in = 4 * size, step = gated ? 2 * size : 4 * size;  // the widest accesses' bytes
  p.wide = sg::aligned(base, in) && sg::aligned(out, step) &&
           (m == 1 || (p.ldb * size % in == 0 && ldo * size % step == 0));
  // What TMA can read and write: rows that start on 16 bytes.
  auto rows_of_16 = [&](const void* b, long long ld) {
    return sg::aligned(b, 16) && (m == 1 || ld * size % 16 == 0);
  };
  p.out_tma = rows_of_16(out, ldo);
  p.base_tma = (base || epi == STRASGPT_EPI_ADD) && (!base || rows_of_16(base, ldb)) &&
               (epi != STRASGPT_EPI_ADD || p.out_tma);
  p.tokens = tokens_of(m, rank, adapters, sms);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = type == STRASGPT_F32 ? launch_type<float>(p, dev, sms, s)
                                             : launch_type<uint16_t>(p, dev, sms, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}
