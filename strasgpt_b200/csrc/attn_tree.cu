// strasgpt_k_attn_tree: GQA attention of a tree of drafted tokens over the
// cache that ends with the tree's own rows.
//
// Drafted token i and head h attend to the cached keys 0..n-1 and to the
// drafted keys j (cache row n + j) whose bit j is set in row i of the mask:
//   s = q.k / sqrt(head_dim),  att = sum exp(s) v / sum exp(s).
//
// All rows (i, h) of a kv head read the same cache, so a CTA takes 16, 32, 64
// or 128 of them as the rows of matrix instructions and walks a share of the
// keys, tile by tile, with the running maximum, sum and output of each row in
// registers (one pass over the cache). The keys are split over as many CTAs
// as fill the GPU; k_merge joins their parts.
//
// fp32 operands keep 21 bits or more: each is the sum of two tf32 values (the
// upper 19 bits and what they leave), and a product takes three tf32 MMAs
// (hi.hi + hi.lo + lo.hi). The bf16 form multiplies its inputs as they are
// and carries the probabilities as two bf16 parts, so that the only rounding
// to bf16 is that of the result.
//
// What bounds it: the cache's bytes with up to 16 rows a kv head in bf16 (90
// us for 8 heads of 128000 keys of 128 entries, 5.8 TB/s) and up to 4 in fp32
// (190 us, 5.5 TB/s, by FMAs: k_tree_few); mma.sync in fp32 with 16 (244 us:
// its three products take 174 us of that, as the slope from 32 to 64 rows
// says) and above; from 17 or 33 rows on the cached keys are attn_tree_tc.cu's
// (see on_tc). Short caches are latency: 7.4 us for one token over 613 keys,
// both kernels.
#include "attn_tree.h"

#include <limits.h>
#include <math.h>

#include <algorithm>

extern "C" {
#include "strasgpt_kernels.h"
}

namespace {

typedef unsigned long long u64;

constexpr int kStages = 3;       // key/value tiles in flight
constexpr int kMaxSplits = 256;

using sg::TreeArgs;

__device__ __forceinline__ uint32_t saddr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo with hi its upper 19 bits (a tf32 value) and lo the exact
// remainder cut to tf32: 21 bits of x at least.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xFFFFE000u;
}
// Two values -> their bf16 halves (x0 in the low 16 bits) and the bf16 of
// what those leave.
__device__ __forceinline__ void split_bf16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(x1), "f"(x0));
  const float r0 = x0 - __uint_as_float(hi << 16);
  const float r1 = x1 - __uint_as_float(hi & 0xFFFF0000u);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(r1), "f"(r0));
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ bool finite4(float4 v) {
  return finite(v.x) && finite(v.y) && finite(v.z) && finite(v.w);
}
__device__ __forceinline__ bool finite_bf16x8(uint4 v) {
  bool ok = true;
  for (uint32_t w : {v.x, v.y, v.z, v.w})
    ok = ok && (w & 0x7F80u) != 0x7F80u && (w & 0x7F800000u) != 0x7F800000u;
  return ok;
}

// Keys of a tile and the padded rows in which it lies in shared memory. The
// paddings make every fragment load below free of bank conflicts: 16 bytes
// shift ldmatrix rows (bf16) and the fp32 value rows 2c apart by two 16-byte
// groups; 64 bytes put neighbouring fp32 key rows on opposite banks.
//
// CTAs of up to four warps are two to an SM, and their tiles must leave room:
// with head_dim 32, where a row's padding is as much as half of it, that takes
// half the keys (16 rows over 8 x 128000 keys: fp32 92 -> 85 us, bf16 54 -> 54;
// over 8 x 4000: 11.0 -> 9.2, 8.4 -> 7.9). Larger CTAs have an SM each.
constexpr size_t kSmSmem = 228 * 1024, kCtaReserved = 1024;

template <typename T, int HD, int WARPS>
struct Tile {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kKeys = (kF32 ? 4096 : 8192) / HD / (WARPS <= 4 && HD == 32 ? 2 : 1);
  static constexpr int kKRow = HD * (int)sizeof(T) + (kF32 ? 64 : 16);
  static constexpr int kVRow = HD * (int)sizeof(T) + 16;
  static constexpr int kStage = kKeys * (kKRow + kVRow);
  static constexpr size_t kBytes = (size_t)kStages * kStage;
  static_assert((WARPS <= 4 ? 2 : 1) * (kBytes + kCtaReserved) <= kSmSmem, "the CTAs of an SM fit");
};

// The tiles of a split: the cached keys, then the drafted ones. A tile holds
// keys of one kind, never of both.
template <typename T, int HD, int THREADS>
struct Walk {
  using L = Tile<T, HD, THREADS / 32>;
  const T *k, *v;                // of the kv head
  int t, n, old_tiles, tile0, tile1;
  uint32_t smem;

  // The cache's length is read on the device (a captured call serves every
  // later length); one outside the cache is cut to it.
  __device__ Walk(const TreeArgs& a, int split, int head, const void* stages) {
    t = a.t;
    n = sg::tree_cached(a);
    old_tiles = (n + L::kKeys - 1) / L::kKeys;
    const int tiles = old_tiles + (t + L::kKeys - 1) / L::kKeys;
    const int per = (tiles + a.splits - 1) / a.splits;
    tile0 = split * per;
    tile1 = min(tiles, tile0 + per);
    k = static_cast<const T*>(a.k) + (size_t)head * a.ctx * HD;
    v = static_cast<const T*>(a.v) + (size_t)head * a.ctx * HD;
    smem = saddr(stages);
  }
  // First cache row of a tile and its rows.
  __device__ void extent(int tile, int& row, int& rows) const {
    const bool old = tile < old_tiles;
    const int k0 = (old ? tile : tile - old_tiles) * L::kKeys;
    row = old ? k0 : n + k0;
    rows = min(L::kKeys, (old ? n : t) - k0);
  }
  __device__ void fetch(int tile) const {
    if (tile < tile1) {
      int row, rows;
      extent(tile, row, rows);
      const uint32_t ks = smem + (tile - tile0) % kStages * L::kStage;
      const uint32_t vs = ks + L::kKeys * L::kKRow;
      constexpr int kVecs = HD * (int)sizeof(T) / 16;
#pragma unroll 8
      for (int i = threadIdx.x; i < L::kKeys * kVecs; i += THREADS) {
        const int r = i / kVecs, x = i % kVecs;
        const int bytes = r < rows ? 16 : 0;  // rows behind the last key are zeros
        const size_t at = (size_t)(row + (r < rows ? r : 0)) * HD + x * (16 / sizeof(T));
        cp_async16(ks + r * L::kKRow + x * 16, k + at, bytes);
        cp_async16(vs + r * L::kVRow + x * 16, v + at, bytes);
      }
    }
    cp_async_commit();
  }
};

// MW warps side by side in rows (16 each), KW in keys.
template <typename T, int HD, int MW, int KW>
__global__ void __launch_bounds__(32 * MW * KW, MW* KW <= 4 ? 2 : 1) k_tree(TreeArgs a) {
  using L = Tile<T, HD, MW * KW>;
  constexpr bool kF32 = L::kF32;
  constexpr int kThreads = 32 * MW * KW;
  constexpr int kRows = 16 * MW;
  constexpr int kKeys = L::kKeys, kWarpKeys = kKeys / KW;
  constexpr int kChunk = kWarpKeys < 32 ? kWarpKeys : 32;  // keys per softmax step of a warp
  constexpr int kN8 = kChunk / 8;
  constexpr int kOut = HD / 8;  // n8 tiles of the output
  static_assert(kChunk % (kF32 ? 8 : 16) == 0, "a warp's keys fill k steps");
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
  const int mw = warp % MW, kw = warp / MW;
  const int split = blockIdx.x, head = blockIdx.y, r0 = blockIdx.z * kRows;
  const int R = a.t * a.group;
  sg::pdl_trigger();
  sg::pdl_wait();

  const Walk<T, HD, kThreads> walk(a, split, head, smem);
  const int n = walk.n, old_tiles = walk.old_tiles, tile0 = walk.tile0, tile1 = walk.tile1;
  if (tile0 >= tile1) return;
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) walk.fetch(tile0 + s);

  // This lane's rows g8 and g8 + 8 of the warp's 16.
  const int rA = r0 + 16 * mw + g8, rB = rA + 8;
  const int tA = rA / a.group, tB = rB / a.group;
  const bool inA = rA < R, inB = rB < R;
  const T* qA = static_cast<const T*>(a.q) + (inA ? tA : 0) * a.ldq +
                (size_t)(head * a.group + (inA ? rA - tA * a.group : 0)) * HD;
  const T* qB = static_cast<const T*>(a.q) + (inB ? tB : 0) * a.ldq +
                (size_t)(head * a.group + (inB ? rB - tB * a.group : 0)) * HD;
  // Scores in units of log2, so that the softmax is exp2.
  const float scale = 1.4426950408889634f / sqrtf((float)HD);

  // Queries as A operands. fp32: raw values, 16 entries of the head per step;
  // slots (c, c + 4) of its two k8 steps hold entries 4c, 4c+1 and 4c+2, 4c+3
  // (keys are read in the same order, so one float4 feeds both steps).
  // bf16: the fragment of m16n8k16.
  constexpr int kQ = HD / 16;
  float4 q4[kF32 ? kQ : 1][2];
  uint32_t q16[kF32 ? 1 : kQ][4];
#pragma unroll
  for (int j = 0; j < kQ; j++) {
    if constexpr (kF32) {
      auto load = [&](const T* p, bool in) {
        float4 v = *reinterpret_cast<const float4*>(p + 16 * j + 4 * c4);
        return in ? make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale)
                  : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      q4[j][0] = load(qA, inA);
      q4[j][1] = load(qB, inB);
    } else {
      auto load = [&](const T* p, bool in, int at) {
        return in ? *reinterpret_cast<const uint32_t*>(p + 16 * j + at) : 0u;
      };
      q16[j][0] = load(qA, inA, 2 * c4);
      q16[j][1] = load(qB, inB, 2 * c4);
      q16[j][2] = load(qA, inA, 2 * c4 + 8);
      q16[j][3] = load(qB, inB, 2 * c4 + 8);
    }
  }

  // Output accumulators. fp32: n8 tile 4b + i holds head entries
  // 32b + 4 column + i (one float4 of a value row feeds four tiles).
  float o[kOut][4];
#pragma unroll
  for (int i = 0; i < kOut; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;

  for (int tile = tile0; tile < tile1; tile++) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    walk.fetch(tile + kStages - 1);  // into the buffer that the last tile left
    int row, rows;
    walk.extent(tile, row, rows);
    const bool old = tile < old_tiles;
    const unsigned char* ks = smem + (tile - tile0) % kStages * L::kStage;
    const unsigned char* vs = ks + kKeys * L::kKRow;
    // A drafted value row with an infinity or NaN may be hidden from some of
    // the rows: 0 * NaN in a matrix instruction would reach them. Such a tile
    // takes the slow product below. (Cached rows are seen by all.)
    bool slow = false;
    if (!old) {
      bool bad = false;
      constexpr int kVecs = HD * (int)sizeof(T) / 16;
      for (int i = threadIdx.x; i < kKeys * kVecs; i += kThreads) {
        const unsigned char* p = vs + i / kVecs * L::kVRow + i % kVecs * 16;
        if constexpr (kF32)
          bad = bad || !finite4(*reinterpret_cast<const float4*>(p));
        else
          bad = bad || !finite_bf16x8(*reinterpret_cast<const uint4*>(p));
      }
      slow = __syncthreads_or(bad);
    }

#pragma unroll 1
    for (int ch = 0; ch < kWarpKeys; ch += kChunk) {
      const int k0 = kw * kWarpKeys + ch;  // first key of the chunk in the tile
      if (k0 >= rows) break;
      float s[kN8][4];
#pragma unroll
      for (int i = 0; i < kN8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
      if constexpr (kF32) {
        // The tensor cores cut their sums: 16 entries at a time from zero,
        // small products first, then added with rounding.
        const unsigned char* kp = ks + (k0 + g8) * L::kKRow + c4 * 16;
#pragma unroll
        for (int j = 0; j < kQ; j++) {
          uint32_t ah[2][4], al[2][4];
          split_tf32(q4[j][0].x, ah[0][0], al[0][0]);
          split_tf32(q4[j][1].x, ah[0][1], al[0][1]);
          split_tf32(q4[j][0].y, ah[0][2], al[0][2]);
          split_tf32(q4[j][1].y, ah[0][3], al[0][3]);
          split_tf32(q4[j][0].z, ah[1][0], al[1][0]);
          split_tf32(q4[j][1].z, ah[1][1], al[1][1]);
          split_tf32(q4[j][0].w, ah[1][2], al[1][2]);
          split_tf32(q4[j][1].w, ah[1][3], al[1][3]);
#pragma unroll
          for (int i = 0; i < kN8; i++) {
            const float4 kv = *reinterpret_cast<const float4*>(kp + i * 8 * L::kKRow + j * 64);
            uint32_t bh[4], bl[4];
            split_tf32(kv.x, bh[0], bl[0]);
            split_tf32(kv.y, bh[1], bl[1]);
            split_tf32(kv.z, bh[2], bl[2]);
            split_tf32(kv.w, bh[3], bl[3]);
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            mma_tf32(x, ah[0], bl[0], bl[1]);
            mma_tf32(y, ah[1], bl[2], bl[3]);
            mma_tf32(x, al[0], bh[0], bh[1]);
            mma_tf32(y, al[1], bh[2], bh[3]);
            mma_tf32(x, ah[0], bh[0], bh[1]);
            mma_tf32(y, ah[1], bh[2], bh[3]);
#pragma unroll
            for (int e = 0; e < 4; e++) s[i][e] += x[e] + y[e];
          }
        }
      } else {
        const uint32_t kp = saddr(ks) + (k0 + (lane & 7) + (lane >> 4) * 8) * L::kKRow +
                            ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int j = 0; j < kQ; j++)
#pragma unroll
          for (int i = 0; i < kN8; i += 2) {
            uint32_t b[4];
            ldsm4(kp + i * 8 * L::kKRow + j * 32, b);
            mma_bf16(s[i], q16[j], b[0], b[1]);
            mma_bf16(s[i + 1], q16[j], b[2], b[3]);
          }
#pragma unroll
        for (int i = 0; i < kN8; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[i][e] *= scale;
      }

      // What the rows may see: all cached keys, or the mask's bits.
      if (!old) {
        const int j0 = row - n + k0;  // drafted index, a multiple of 8
        const u64 wA = inA ? a.mask[(size_t)tA * a.words + (j0 >> 6)] >> (j0 & 63) : 0;
        const u64 wB = inB ? a.mask[(size_t)tB * a.words + (j0 >> 6)] >> (j0 & 63) : 0;
#pragma unroll
        for (int i = 0; i < kN8; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int j = 8 * i + 2 * c4 + e;
            const bool in = k0 + j < rows;
            if (!(in && (wA >> j & 1))) s[i][e] = -INFINITY;
            if (!(in && (wB >> j & 1))) s[i][2 + e] = -INFINITY;
          }
      } else if (k0 + kChunk > rows) {
#pragma unroll
        for (int i = 0; i < kN8; i++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (k0 + 8 * i + 2 * c4 + e >= rows) s[i][e] = s[i][2 + e] = -INFINITY;
      }

      // Online softmax; the four lanes of a row share its keys.
      float xA = -INFINITY, xB = -INFINITY;
#pragma unroll
      for (int i = 0; i < kN8; i++) {
        xA = fmaxf(xA, fmaxf(s[i][0], s[i][1]));
        xB = fmaxf(xB, fmaxf(s[i][2], s[i][3]));
      }
      xA = fmaxf(xA, __shfl_xor_sync(0xFFFFFFFFu, xA, 1));
      xA = fmaxf(xA, __shfl_xor_sync(0xFFFFFFFFu, xA, 2));
      xB = fmaxf(xB, __shfl_xor_sync(0xFFFFFFFFu, xB, 1));
      xB = fmaxf(xB, __shfl_xor_sync(0xFFFFFFFFu, xB, 2));
      const float nA = fmaxf(mA, xA), nB = fmaxf(mB, xB);
      if (__any_sync(0xFFFFFFFFu, nA > mA || nB > mB)) {
        // A row that has seen no key yet keeps m = -inf and zeros.
        const float fA = nA == -INFINITY ? 1.f : exp2f(mA - nA);
        const float fB = nB == -INFINITY ? 1.f : exp2f(mB - nB);
        mA = nA;
        mB = nB;
        lA *= fA;
        lB *= fB;
#pragma unroll
        for (int i = 0; i < kOut; i++) {
          o[i][0] *= fA;
          o[i][1] *= fA;
          o[i][2] *= fB;
          o[i][3] *= fB;
        }
      }
      const float zA = mA == -INFINITY ? 0.f : mA, zB = mB == -INFINITY ? 0.f : mB;
#pragma unroll
      for (int i = 0; i < kN8; i++) {
        s[i][0] = exp2f(s[i][0] - zA);
        s[i][1] = exp2f(s[i][1] - zA);
        s[i][2] = exp2f(s[i][2] - zB);
        s[i][3] = exp2f(s[i][3] - zB);
        lA += s[i][0] + s[i][1];
        lB += s[i][2] + s[i][3];
      }

      if (slow) {
        // Key by key, weights of exactly 0 left out.
        for (int kk = 0; kk < kChunk && k0 + kk < rows; kk++) {
          float pA = 0.f, pB = 0.f;
#pragma unroll
          for (int i = 0; i < kN8; i++)
            if (i == kk / 8) {
              pA = kk & 1 ? s[i][1] : s[i][0];
              pB = kk & 1 ? s[i][3] : s[i][2];
            }
          const int from = (lane & ~3) | (kk % 8 / 2);
          pA = __shfl_sync(0xFFFFFFFFu, pA, from);
          pB = __shfl_sync(0xFFFFFFFFu, pB, from);
          const T* vr = reinterpret_cast<const T*>(vs + (k0 + kk) * L::kVRow);
#pragma unroll
          for (int i = 0; i < kOut; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float v;
              if constexpr (kF32)
                v = vr[32 * (i / 4) + 4 * (2 * c4 + e) + i % 4];
              else
                v = sg::bf16_to_f32(vr[8 * i + 2 * c4 + e]);
              if (pA != 0.f) o[i][e] += pA * v;
              if (pB != 0.f) o[i][2 + e] += pB * v;
            }
        }
        continue;
      }

      if constexpr (kF32) {
        // The score accumulators are the A operand as they lie: slots c and
        // c + 4 of a k8 step are keys 2c and 2c + 1. A chunk's products are
        // summed from zero and then added, as above.
        uint32_t ph[kN8][4], pl[kN8][4];
#pragma unroll
        for (int i = 0; i < kN8; i++) {
          split_tf32(s[i][0], ph[i][0], pl[i][0]);
          split_tf32(s[i][2], ph[i][1], pl[i][1]);
          split_tf32(s[i][1], ph[i][2], pl[i][2]);
          split_tf32(s[i][3], ph[i][3], pl[i][3]);
        }
        const unsigned char* vp = vs + (k0 + 2 * c4) * L::kVRow + g8 * 16;
#pragma unroll
        for (int b = 0; b < HD / 32; b++) {
          float x[4][4];
#pragma unroll
          for (int e = 0; e < 4; e++) x[e][0] = x[e][1] = x[e][2] = x[e][3] = 0.f;
#pragma unroll
          for (int i = 0; i < kN8; i++) {
            const float4 v0 =
                *reinterpret_cast<const float4*>(vp + i * 8 * L::kVRow + b * 128);
            const float4 v1 =
                *reinterpret_cast<const float4*>(vp + (i * 8 + 1) * L::kVRow + b * 128);
            uint32_t h0[4], l0[4], h1[4], l1[4];
            split_tf32(v0.x, h0[0], l0[0]);
            split_tf32(v0.y, h0[1], l0[1]);
            split_tf32(v0.z, h0[2], l0[2]);
            split_tf32(v0.w, h0[3], l0[3]);
            split_tf32(v1.x, h1[0], l1[0]);
            split_tf32(v1.y, h1[1], l1[1]);
            split_tf32(v1.z, h1[2], l1[2]);
            split_tf32(v1.w, h1[3], l1[3]);
#pragma unroll
            for (int e = 0; e < 4; e++) mma_tf32(x[e], ph[i], l0[e], l1[e]);
#pragma unroll
            for (int e = 0; e < 4; e++) mma_tf32(x[e], pl[i], h0[e], h1[e]);
#pragma unroll
            for (int e = 0; e < 4; e++) mma_tf32(x[e], ph[i], h0[e], h1[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int y = 0; y < 4; y++) o[4 * b + e][y] += x[e][y];
        }
      } else {
        const uint32_t vp = saddr(vs) + (k0 + (lane & 7) + ((lane >> 3) & 1) * 8) * L::kVRow +
                            (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < kN8; i += 2) {
          uint32_t ph[4], pl[4];
          split_bf16(s[i][0], s[i][1], ph[0], pl[0]);
          split_bf16(s[i][2], s[i][3], ph[1], pl[1]);
          split_bf16(s[i + 1][0], s[i + 1][1], ph[2], pl[2]);
          split_bf16(s[i + 1][2], s[i + 1][3], ph[3], pl[3]);
#pragma unroll
          for (int b = 0; b < kOut; b += 2) {
            uint32_t v[4];
            ldsm4t(vp + i * 8 * L::kVRow + b * 16, v);
            mma_bf16(o[b], ph, v[0], v[1]);
            mma_bf16(o[b + 1], ph, v[2], v[3]);
            mma_bf16(o[b], pl, v[0], v[1]);
            mma_bf16(o[b + 1], pl, v[2], v[3]);
          }
        }
      }
    }
  }
  cp_async_wait<0>();
  lA += __shfl_xor_sync(0xFFFFFFFFu, lA, 1);
  lA += __shfl_xor_sync(0xFFFFFFFFu, lA, 2);
  lB += __shfl_xor_sync(0xFFFFFFFFu, lB, 1);
  lB += __shfl_xor_sync(0xFFFFFFFFu, lB, 2);

  // The key warps' parts of the rows are joined in shared memory, warps of
  // the upper half into the lower one.
  if constexpr (KW > 1) {
    constexpr int kLane = kOut * 4 + 4;  // values a lane hands over
    float* x = reinterpret_cast<float*>(smem);
    static_assert((size_t)MW * (KW / 2) * 32 * kLane * 4 <= L::kBytes, "join fits the tiles");
#pragma unroll
    for (int half = KW / 2; half > 0; half /= 2) {
      __syncthreads();
      // [value][warp][lane]: lanes side by side.
      if (kw >= half && kw < 2 * half) {
        float* p = x + ((kw - half) * MW + mw) * 32 + lane;
        constexpr int kStep = MW * (KW / 2) * 32;
#pragma unroll
        for (int i = 0; i < kOut; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) p[(4 * i + e) * kStep] = o[i][e];
        p[(4 * kOut) * kStep] = mA;
        p[(4 * kOut + 1) * kStep] = mB;
        p[(4 * kOut + 2) * kStep] = lA;
        p[(4 * kOut + 3) * kStep] = lB;
      }
      __syncthreads();
      if (kw < half) {
        const float* p = x + (kw * MW + mw) * 32 + lane;
        constexpr int kStep = MW * (KW / 2) * 32;
        const float m2A = p[(4 * kOut) * kStep], m2B = p[(4 * kOut + 1) * kStep];
        const float nA = fmaxf(mA, m2A), nB = fmaxf(mB, m2B);
        const float fA = nA == -INFINITY ? 0.f : exp2f(mA - nA);
        const float fB = nB == -INFINITY ? 0.f : exp2f(mB - nB);
        const float gA = nA == -INFINITY ? 0.f : exp2f(m2A - nA);
        const float gB = nB == -INFINITY ? 0.f : exp2f(m2B - nB);
        lA = lA * fA + p[(4 * kOut + 2) * kStep] * gA;
        lB = lB * fB + p[(4 * kOut + 3) * kStep] * gB;
        mA = nA;
        mB = nB;
#pragma unroll
        for (int i = 0; i < kOut; i++) {
          o[i][0] = o[i][0] * fA + p[(4 * i) * kStep] * gA;
          o[i][1] = o[i][1] * fA + p[(4 * i + 1) * kStep] * gA;
          o[i][2] = o[i][2] * fB + p[(4 * i + 2) * kStep] * gB;
          o[i][3] = o[i][3] * fB + p[(4 * i + 3) * kStep] * gB;
        }
      }
    }
    if (kw > 0) return;
  }

  // One split: the rows are complete (a row without keys is zeros). Else the
  // parts go to the workspace as they are, in 32 bits.
  const bool whole = a.splits == 1;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int r = half ? rB : rA, tok = half ? tB : tA;
    if (r >= R) continue;
    const float m = half ? mB : mA, l = half ? lB : lA;
    const float f = whole ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
    const size_t at = ((size_t)split * a.kh + head) * R + r;
    if (!whole && c4 == 0) a.ml[at] = make_float2(m, l);
    T* out = static_cast<T*>(a.att) + tok * a.ldo +
             (size_t)(head * a.group + r - tok * a.group) * HD;
    float* part = a.part + at * HD;
    if constexpr (kF32) {
      float* to = whole ? reinterpret_cast<float*>(out) : part;
#pragma unroll
      for (int b = 0; b < HD / 32; b++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          *reinterpret_cast<float4*>(to + 32 * b + 8 * c4 + 4 * e) =
              make_float4(o[4 * b][2 * half + e] * f, o[4 * b + 1][2 * half + e] * f,
                          o[4 * b + 2][2 * half + e] * f, o[4 * b + 3][2 * half + e] * f);
    } else {
#pragma unroll
      for (int i = 0; i < kOut; i++) {
        const float x0 = o[i][2 * half] * f, x1 = o[i][2 * half + 1] * f;
        if (whole) {
          uint32_t w;
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(x1), "f"(x0));
          *reinterpret_cast<uint32_t*>(out + 8 * i + 2 * c4) = w;
        } else {
          *reinterpret_cast<float2*>(part + 8 * i + 2 * c4) = make_float2(x0, x1);
        }
      }
    }
  }
}

// Up to kFewRows rows a kv head, fp32, head_dim 128: FMAs. Most of a matrix
// instruction's 16 rows would be empty, and three products of each bound
// k_tree: 4 rows over 8 x 128000 keys take 238 us there, 190 here (5.5 TB/s),
// over 8 x 500 9.4 and 7.9. (With shorter heads a key's softmax outweighs its
// products: 64 entries 111 there, 128 here.) A warp takes 8 keys at a time;
// four lanes share a key's scores, each having a quarter of the entries of key
// and queries, then every lane has 4 entries of the outputs.
constexpr int kFewRows = 4, kFewWarps = 4, kFewHeadDim = 128;

__global__ void __launch_bounds__(32 * kFewWarps, 2) k_tree_few(TreeArgs a) {
  constexpr int HD = kFewHeadDim;
  using L = Tile<float, HD, kFewWarps>;
  constexpr int kWarpKeys = L::kKeys / kFewWarps, kQ = HD / 16, kO = HD / 32;
  static_assert(kWarpKeys == 8, "a warp's keys of a tile are one step");
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
  const int split = blockIdx.x, head = blockIdx.y, R = a.t * a.group;
  sg::pdl_trigger();
  sg::pdl_wait();
  const Walk<float, HD, 32 * kFewWarps> walk(a, split, head, smem);
  if (walk.tile0 >= walk.tile1) return;
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) walk.fetch(walk.tile0 + s);

  // Scores in units of log2, so that the softmax is exp2.
  const float scale = 1.4426950408889634f / sqrtf((float)HD);
  float4 q[kFewRows][kQ];
  float m[kFewRows], l[kFewRows], o[kFewRows][kO];
#pragma unroll
  for (int r = 0; r < kFewRows; r++) {
    const int row = r < R ? r : 0, tok = row / a.group;
    const float* from = static_cast<const float*>(a.q) + tok * a.ldq +
                        (size_t)(head * a.group + row - tok * a.group) * HD + 4 * c4;
#pragma unroll
    for (int j = 0; j < kQ; j++) {
      q[r][j] = *reinterpret_cast<const float4*>(from + 16 * j);
      q[r][j].x *= scale;
      q[r][j].y *= scale;
      q[r][j].z *= scale;
      q[r][j].w *= scale;
    }
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kO; i++) o[r][i] = 0.f;
  }

  for (int tile = walk.tile0; tile < walk.tile1; tile++) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    walk.fetch(tile + kStages - 1);  // into the buffer that the last tile left
    int row, rows;
    walk.extent(tile, row, rows);
    const bool old = tile < walk.old_tiles;
    const unsigned char* ks = smem + (tile - walk.tile0) % kStages * L::kStage;
    const unsigned char* vs = ks + L::kKeys * L::kKRow;
    const int k0 = warp * kWarpKeys;  // the warp's first key in the tile
    if (k0 < rows) {
      float s[kFewRows][2];
#pragma unroll
      for (int r = 0; r < kFewRows; r++) s[r][0] = s[r][1] = 0.f;
      const unsigned char* kp = ks + (k0 + g8) * L::kKRow + c4 * 16;
#pragma unroll
      for (int j = 0; j < kQ; j++) {
        const float4 x = *reinterpret_cast<const float4*>(kp + j * 64);
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
          s[r][0] = fmaf(q[r][j].x, x.x, s[r][0]);
          s[r][1] = fmaf(q[r][j].y, x.y, s[r][1]);
          s[r][0] = fmaf(q[r][j].z, x.z, s[r][0]);
          s[r][1] = fmaf(q[r][j].w, x.w, s[r][1]);
        }
      }
      float p[kFewRows], top[kFewRows];
#pragma unroll
      for (int r = 0; r < kFewRows; r++) {
        p[r] = s[r][0] + s[r][1];
        p[r] += __shfl_xor_sync(0xFFFFFFFFu, p[r], 1);
        p[r] += __shfl_xor_sync(0xFFFFFFFFu, p[r], 2);
        bool in = k0 + g8 < rows && r < R;
        if (!old && in) {
          const int j = row - walk.n + k0 + g8;  // drafted index
          in = a.mask[(size_t)(r / a.group) * a.words + (j >> 6)] >> (j & 63) & 1;
        }
        if (!in) p[r] = -INFINITY;
        top[r] = fmaxf(p[r], __shfl_xor_sync(0xFFFFFFFFu, p[r], 4));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 8));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 16));
      }
#pragma unroll
      for (int r = 0; r < kFewRows; r++) {
        if (top[r] > m[r]) {  // the same in all lanes
          const float f = exp2f(m[r] - top[r]);
          m[r] = top[r];
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < kO; i++) o[r][i] *= f;
        }
        // A row that has seen no key yet keeps m = -inf and zeros.
        p[r] = exp2f(p[r] - (m[r] == -INFINITY ? 0.f : m[r]));
        l[r] += p[r];
      }
      const unsigned char* vp = vs + k0 * L::kVRow + lane * kO * 4;
#pragma unroll
      for (int kk = 0; kk < 8; kk++) {
        const float4 v4 = *reinterpret_cast<const float4*>(vp + kk * L::kVRow);
        const float x[kO] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
          const float w = __shfl_sync(0xFFFFFFFFu, p[r], 4 * kk);
          // A drafted row that is hidden may hold anything; cached ones are
          // seen by all.
          if (old || w != 0.f) {
#pragma unroll
            for (int i = 0; i < kO; i++) o[r][i] = fmaf(w, x[i], o[r][i]);
          }
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // The warps' parts are joined in shared memory, a row by each warp.
  float* part = reinterpret_cast<float*>(smem);  // [warp][row][HD + 2]
  static_assert(kFewWarps * kFewRows * (HD + 2) * 4 <= (int)L::kBytes, "join fits the tiles");
  static_assert(kFewWarps == kFewRows, "a warp per row");
#pragma unroll
  for (int r = 0; r < kFewRows; r++) {
    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 4);
    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 8);
    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 16);
    float* to = part + (warp * kFewRows + r) * (HD + 2);
#pragma unroll
    for (int i = 0; i < kO; i++) to[lane * kO + i] = o[r][i];
    if (lane == 0) {
      to[HD] = m[r];
      to[HD + 1] = l[r];
    }
  }
  __syncthreads();
  if (warp >= R) return;
  float all = -INFINITY, sum = 0.f, out[kO];
#pragma unroll
  for (int i = 0; i < kO; i++) out[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kFewWarps; w++)
    all = fmaxf(all, part[(w * kFewRows + warp) * (HD + 2) + HD]);
#pragma unroll
  for (int w = 0; w < kFewWarps; w++) {
    const float* from = part + (w * kFewRows + warp) * (HD + 2);
    const float f = all == -INFINITY ? 0.f : exp2f(from[HD] - all);
    sum += from[HD + 1] * f;
#pragma unroll
    for (int i = 0; i < kO; i++) out[i] = fmaf(from[lane * kO + i], f, out[i]);
  }
  // One split: the row is complete (one without keys is zeros). Else its part
  // goes to the workspace.
  const bool whole = a.splits == 1;
  const float f = whole ? (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)) : 1.f;
  const int tok = warp / a.group;
  const size_t at = ((size_t)split * a.kh + head) * R + warp;
  if (!whole && lane == 0) a.ml[at] = make_float2(all, sum);
  float* to = whole ? static_cast<float*>(a.att) + tok * a.ldo +
                          (size_t)(head * a.group + warp - tok * a.group) * HD
                    : a.part + at * HD;
#pragma unroll
  for (int i = 0; i < kO; i++) to[lane * kO + i] = out[i] * f;
}

// A block joins the parts of one row: sixteen groups of eight lanes, a lane
// having HD / 8 entries of the head, take the parts in turn, each with a
// running maximum of its own, so that a row's loads are all on their way at
// once; then the groups are joined.
//
// DRAFTED: the parts have the cached keys only. The drafted ones that the row
// sees, its ancestors in the tree and itself, come first, a group per key: a
// few keys as a rule, for which a matrix tile would be nearly empty, and rows
// it does not see are not even read.
constexpr int kMergeThreads = 128, kMergeGroups = kMergeThreads / 8;

template <typename T, int HD, bool DRAFTED>
__global__ void __launch_bounds__(kMergeThreads) k_merge(TreeArgs a, int keys_per_tile) {
  constexpr int V = HD / 8;  // entries per lane
  constexpr bool kF32 = sizeof(T) == 4;
  __shared__ float warp_o[kMergeThreads / 32][HD];
  __shared__ float2 warp_ml[kMergeThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = threadIdx.x >> 3, e0 = (threadIdx.x & 7) * V;
  const int R = a.t * a.group, row = blockIdx.x;
  sg::pdl_trigger();
  sg::pdl_wait();
  const int n = sg::tree_cached(a);
  const int tiles = (n + keys_per_tile - 1) / keys_per_tile +
                    (DRAFTED ? 0 : (a.t + keys_per_tile - 1) / keys_per_tile);
  const int per = (tiles + a.splits - 1) / a.splits;
  const int parts = tiles ? (tiles + per - 1) / per : 0;
  const int head = row / R, r = row - head * R, tok = r / a.group;
  const size_t at = (size_t)(head * a.group + r - tok * a.group) * HD;
  auto read = [&](const T* p, float* x) {
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + i);
        x[i] = sg::bf16_lo(v.x); x[i + 1] = sg::bf16_hi(v.x);
        x[i + 2] = sg::bf16_lo(v.y); x[i + 3] = sg::bf16_hi(v.y);
      }
    }
  };
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; i++) o[i] = 0.f;
  // Adds outputs x with maximum and sum (m2, l2).
  auto join = [&](float m2, float l2, const float* x) {
    const float next = fmaxf(m, m2);
    const float f = next == -INFINITY ? 1.f : exp2f(m - next);
    const float g = next == -INFINITY ? 1.f : exp2f(m2 - next);
    m = next;
    l = l * f + l2 * g;
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = fmaf(x[i], g, o[i] * f);
  };
  if constexpr (DRAFTED) {
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    float q[V];
    read(static_cast<const T*>(a.q) + tok * a.ldq + at + e0, q);
#pragma unroll
    for (int i = 0; i < V; i++) q[i] *= scale;
    const size_t base = ((size_t)head * a.ctx + n) * HD + e0;
    const T* k = static_cast<const T*>(a.k) + base;
    const T* v = static_cast<const T*>(a.v) + base;
    int seen = 0;  // keys in the words before
    for (int w = 0; w < a.words; w++) {
      u64 bits = a.mask[(size_t)tok * a.words + w];
      if (a.t - 64 * w < 64) bits &= (1ull << (a.t - 64 * w)) - 1;
      // This group's keys: those whose number among the row's is the group's,
      // modulo the groups. (Lanes of a warp come out of the loop together.)
      const int count = __popcll(bits);
      int mine = (group - seen % kMergeGroups + kMergeGroups) % kMergeGroups;
      seen += count;
      for (int first = 0; first < count; first += kMergeGroups, mine += kMergeGroups) {
        const bool in = mine < count;
        int j = 0;
        if (in) {  // the mine-th set bit
          u64 b = bits;
          for (int x = 0; x < mine; x++) b &= b - 1;
          j = 64 * w + __ffsll((long long)b) - 1;
        }
        float x[V], s = 0.f;
        if (in) {
          read(k + (size_t)j * HD, x);
#pragma unroll
          for (int i = 0; i < V; i++) s = fmaf(q[i], x[i], s);
          read(v + (size_t)j * HD, x);
        }
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 4);
        // exp2(s - s) is 1, and NaN where the score is: as one part of sum 1.
        // A score of -inf weighs nothing.
        if (in && s != -INFINITY) join(s == s ? s : m, s == s ? 1.f : s, x);
      }
    }
  }
  const size_t step = (size_t)a.kh * R;
#pragma unroll 2
  for (int s = group; s < parts; s += kMergeGroups) {
    const float2 p = a.ml[s * step + row];
    const float* from = a.part + (s * step + row) * HD + e0;
    float x[V];
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 y = *reinterpret_cast<const float4*>(from + i);
      x[i] = y.x; x[i + 1] = y.y; x[i + 2] = y.z; x[i + 3] = y.w;
    }
    join(p.x, p.y, x);
  }
  // The warp's four groups, then the warps.
  float top = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
  top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
  const float f = top == -INFINITY ? 1.f : exp2f(m - top);
  l *= f;
#pragma unroll
  for (int i = 0; i < V; i++) o[i] *= f;
#pragma unroll
  for (int d = 8; d < 32; d *= 2) {
    l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
#pragma unroll
    for (int i = 0; i < V; i++) o[i] += __shfl_xor_sync(0xFFFFFFFFu, o[i], d);
  }
  if (lane < 8) {
#pragma unroll
    for (int i = 0; i < V; i++) warp_o[warp][e0 + i] = o[i];
    if (lane == 0) warp_ml[warp] = make_float2(top, l);
  }
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float all = -INFINITY, sum = 0.f, out = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; w++) all = fmaxf(all, warp_ml[w].x);
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; w++) {
    const float g = all == -INFINITY ? 1.f : exp2f(warp_ml[w].x - all);
    sum += warp_ml[w].y * g;
    out += warp_o[w][threadIdx.x] * g;
  }
  // A row without keys is zeros.
  out *= sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  T* to = static_cast<T*>(a.att) + tok * a.ldo + at + threadIdx.x;
  if constexpr (kF32)
    *to = out;
  else
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(*to) : "f"(out));
}

// Rows of a kv head -> warps in rows and in keys.
struct Shape {
  int mw, kw;
};
Shape shape_of(int rows) {
  if (rows <= 16) return {1, 4};
  if (rows <= 32) return {2, 2};
  if (rows <= 64) return {4, 1};
  return {8, 1};
}

// Whether the cached keys go to tcgen05 (attn_tree_tc.cu): where mma.sync, not
// the cache's bytes, is what bounds this file's kernel. Measured with 8 kv
// heads, us here / there:
//   head_dim 128, 16 rows: bf16 128000 keys 92 / 91, 8000 14.0 / 15.6;
//                          fp32 128000 keys 244 / 295, 8000 29 / 32
//                 32 rows: bf16 119 / 93, 19.0 / 16.5; fp32 409 / 301, 40 / 33
//   head_dim 64,  32 rows: bf16 76 / 69, 11.3 / 13.3; fp32 190 / 211, 22 / 23
//                 48 rows: bf16 120 / 69, 14.2 / 13.6; fp32 338 / 212, 32 / 23
// Not for many drafted tokens, whose own keys the merge reads one by one, and
// not for head_dim 32.
bool on_tc(int t, int group, int hd) {
  return t <= 256 && hd >= 64 && t * group > (hd == 128 ? 16 : 32);
}

// Splits of the keys: as many CTAs as the GPU holds at once.
int splits_of(int sms, int t, int kh, int group, int hd) {
  const int rows = t * group;
  const Shape s = shape_of(rows);
  const bool tc = on_tc(t, group, hd);
  const int resident = sms * (!tc && s.mw * s.kw <= 4 ? 2 : 1);
  const int tile = tc ? sg::kTreeTcRows : 16 * s.mw;
  const long long others = (long long)kh * ((rows + tile - 1) / tile);
  return (int)std::max(1ll, std::min((long long)kMaxSplits, resident / others));
}

size_t workspace_of(int splits, int t, int kh, int group, int hd) {
  if (splits == 1 && !on_tc(t, group, hd)) return 0;
  return (size_t)splits * kh * t * group * (hd + 2) * sizeof(float);
}

cudaError_t launch_few(const TreeArgs& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  using L = Tile<float, kFewHeadDim, kFewWarps>;
  cudaError_t e = sg::allow_smem(k_tree_few, L::kBytes, dev, allowed);
  if (e != cudaSuccess) return e;
  e = sg::try_launch(k_tree_few, dim3(a.splits, a.kh), dim3(32 * kFewWarps), L::kBytes, 1, s, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  return sg::try_launch(k_merge<float, kFewHeadDim, false>, dim3(a.t * a.group * a.kh),
                        dim3(kMergeThreads), 0, 1, s, a, L::kKeys);
}

template <typename T, int HD, int MW, int KW>
cudaError_t launch_shape(const TreeArgs& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  using L = Tile<T, HD, MW * KW>;
  constexpr size_t bytes = L::kBytes;
  cudaError_t e = sg::allow_smem(k_tree<T, HD, MW, KW>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  const int rows = a.t * a.group;
  e = sg::try_launch(k_tree<T, HD, MW, KW>,
                     dim3(a.splits, a.kh, (rows + 16 * MW - 1) / (16 * MW)),
                     dim3(32 * MW * KW), bytes, 1, s, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  return sg::try_launch(k_merge<T, HD, false>, dim3(rows * a.kh), dim3(kMergeThreads), 0, 1, s, a,
                        L::kKeys);
}

template <typename T, int HD>
cudaError_t launch_hd(const TreeArgs& a, int dev, cudaStream_t s) {
  if (on_tc(a.t, a.group, HD)) {
    if constexpr (HD >= 64) {
      constexpr bool kF32 = sizeof(T) == 4;
      const cudaError_t e = sg::tree_tc(a, kF32, HD, dev, s);
      if (e != cudaSuccess) return e;
      return sg::try_launch(k_merge<T, HD, true>, dim3(a.t * a.group * a.kh), dim3(kMergeThreads),
                            0, 1, s, a, sg::tree_tc_keys());
    }
  }
  if constexpr (sizeof(T) == 4 && HD == kFewHeadDim)
    if (a.t * a.group <= kFewRows) return launch_few(a, dev, s);
  const Shape f = shape_of(a.t * a.group);
  if (f.mw == 1) return launch_shape<T, HD, 1, 4>(a, dev, s);
  if (f.mw == 2) return launch_shape<T, HD, 2, 2>(a, dev, s);
  if (f.mw == 4) return launch_shape<T, HD, 4, 1>(a, dev, s);
  return launch_shape<T, HD, 8, 1>(a, dev, s);
}

template <typename T>
cudaError_t launch_type(const TreeArgs& a, int hd, int dev, cudaStream_t s) {
  if (hd == 128) return launch_hd<T, 128>(a, dev, s);
  if (hd == 64) return launch_hd<T, 64>(a, dev, s);
  return launch_hd<T, 32>(a, dev, s);
}

const char* bad_shape(int t, int kh, int group, int hd) {
  if (t < 0 || kh <= 0 || group <= 0) return "empty shape";
  if (t > STRASGPT_ATTN_TREE_MAX) return "more than 1024 drafted tokens";
  if (group > 128 || kh > 65535) return "more than 128 q heads per kv head, or 65535 kv heads";
  if (hd != 32 && hd != 64 && hd != 128) return "head_dim must be 32, 64 or 128";
  // k_merge has a block per row.
  if ((long long)t * kh * group > INT_MAX) return "more than 2^31 - 1 rows of q heads";
  return nullptr;
}

}  // namespace

extern "C" {

size_t strasgpt_k_attn_tree_workspace(int t, int kv_heads, int group, int head_dim) {
  const char* const me = "strasgpt_k_attn_tree_workspace";
  if (const char* why = bad_shape(t, kv_heads, group, head_dim)) {
    sg::refuse(me, why);
    return 0;
  }
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) {
    sg::refuse(me, why);
    return 0;
  }
  return t ? workspace_of(splits_of(sms, t, kv_heads, group, head_dim), t, kv_heads, group,
                          head_dim)
           : 0;
}

int strasgpt_k_attn_tree(const void* q, long long ldq, const void* k_cache, const void* v_cache,
                         int type, int t, int kv_heads, int group, int head_dim, int ctx,
                         const int* cached, const uint64_t* mask, void* att, long long ldo,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* const me = "strasgpt_k_attn_tree";
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return sg::refuse(me, "unknown type");
  if (const char* why = bad_shape(t, kv_heads, group, head_dim)) return sg::refuse(me, why);
  if (ctx < t) return sg::refuse(me, "the cache has fewer rows than the tree");
  const long long row = (long long)kv_heads * group * head_dim;
  if (t > 1 && (ldq < row || ldo < row)) return sg::refuse(me, "rows of q or att overlap");
  if (t == 0) return 0;
  if (!q || !k_cache || !v_cache || !cached || !mask || !att)
    return sg::refuse(me, "null buffer");
  const size_t size = type == STRASGPT_F32 ? 4 : 2;
  if (!sg::aligned(q, 16) || !sg::aligned(k_cache, 16) || !sg::aligned(v_cache, 16) ||
      !sg::aligned(att, 16) || (t > 1 && (ldq * size % 16 || ldo * size % 16)))
    return sg::refuse(me, "q, the caches, att and their rows must be 16-byte aligned");
  if (q == att && t > 1 && ldq != ldo)
    return sg::refuse(me, "in place, q and att must have the same strides");
  if (!sg::aligned(cached, 4) || !sg::aligned(mask, 8))
    return sg::refuse(me, "a buffer is not aligned to its entries");
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  for (const void* p : {q, k_cache, v_cache, (const void*)cached, (const void*)mask,
                        (const void*)att})
    if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);
  const int splits = splits_of(sms, t, kv_heads, group, head_dim);
  const size_t need = workspace_of(splits, t, kv_heads, group, head_dim);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return sg::refuse(me, "the workspace is smaller than strasgpt_k_attn_tree_workspace says");
    if (!sg::aligned(workspace, 16)) return sg::refuse(me, "workspace must be 16-byte aligned");
    if (const char* why = sg::not_on_device(workspace, dev)) return sg::refuse(me, why);
  }
  TreeArgs a;
  a.q = q; a.k = k_cache; a.v = v_cache; a.att = att;
  a.ldq = ldq; a.ldo = ldo;
  a.t = t; a.kh = kv_heads; a.group = group; a.ctx = ctx; a.words = (t + 63) / 64;
  a.cached = cached; a.mask = (const u64*)mask;
  a.splits = splits;
  a.part = (float*)workspace;
  a.ml = (float2*)(a.part + (size_t)splits * kv_heads * t * group * head_dim);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = type == STRASGPT_F32 ? launch_type<float>(a, head_dim, dev, s)
                                             : launch_type<uint16_t>(a, head_dim, dev, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}

}  // extern "C"
