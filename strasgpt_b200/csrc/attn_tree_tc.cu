// strasgpt_k_attn_tree, cached keys, for many rows per kv head: tcgen05.
//
// A CTA has 128 rows (drafted token, q head) of one kv head and a share of
// the cached keys, which all of its rows see. Twelve warps: two warpgroups of
// softmax, one thread per row, that take the key tiles in turn; one thread
// that issues the matrix instructions; three warps that bring in keys and
// values. Per tile: S = Q K^T into tensor memory; its warpgroup reads S,
// subtracts the running maximum and writes P = 2^(S - m) over it, as bf16
// parts; O = P V (P read from tensor memory) into tensor memory; the
// warpgroup adds O, scaled, to its registers. Each warpgroup has its own
// maximum, sum and output, joined at the end, so that one's softmax runs
// under the other's matrix instructions and nothing is rescaled in place.
//
// Keys and values lie in shared memory as rows of 64 head entries (128 bytes,
// 128-byte swizzle): K-major for Q K^T, the same rows MN-major for P V.
//
// Precision. bf16: operands as they are, P as two bf16 parts (2^-17). fp32:
// every operand as three bf16 parts, the six products that matter (the others
// are below 2^-24); sums of a tile stay in the tensor cores' fp32, tiles are
// added in registers, rounded to nearest.
//
// Bound: for bf16 with 128 rows the cache's bytes (23 cycles a key at 6.5
// TB/s, against 8 for the matrix instructions and 8 for exp2), with more rows
// the three come together; fp32's six products take 60 cycles a key.
#include "attn_tree.h"

#include <math.h>

namespace sg {
namespace {

constexpr int kRows = kTreeTcRows;
constexpr int kThreads = 384;
constexpr int kLoaders = 96;
constexpr unsigned long long kTimeoutNs = 2000000000ULL;

template <typename T, int HD>
struct Tc {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kParts = kF32 ? 3 : 1;           // of q, k, v
  static constexpr int kPParts = kF32 ? 3 : 2;          // of the probabilities
  static constexpr int kKeys = kF32 ? 64 : 128;
  static constexpr int kQPart = kRows * HD * 2;         // bytes of one part
  static constexpr int kPart = kKeys * HD * 2;
  static constexpr int kTile = kParts * kPart;          // of K, or of V
  // First column of S in its region: P's parts of 32 keys, which overwrite
  // it from the region's start, reach no scores that are still to be read.
  static constexpr int kS = kF32 ? 32 : 0;
  static constexpr int kStages = kF32 ? 1 : 3;
  static constexpr int kLoaded = kF32 ? kLoaders : 32;  // arrivals per filled tile
  // fp32 rows on their way to parts: two buffers of 32 keys.
  static constexpr int kRawKeys = 32;
  static constexpr int kRaw = kF32 ? 2 * kRawKeys * HD * 4 : 0;
  static constexpr int kJoin = kRows * (HD + 4) * 4;    // the warpgroups' join
  static constexpr int kOperands = kParts * kQPart + kStages * 2 * kTile + kRaw;
  static constexpr int kUsed = (kOperands > kJoin ? kOperands : kJoin) + 1024;
  // At least half of an SM's: the CTA has all of the SM's tensor memory.
  static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  // Instruction descriptors: fp32 sums of bf16, M = 128; S: N = keys, both
  // K-major; O: N = head entries, V MN-major.
  static constexpr uint32_t kBase = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t kDescS = kBase | ((uint32_t)(kKeys >> 3) << 17);
  static constexpr uint32_t kDescO = kBase | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
};
// Tensor memory columns: S (then P) and O of each warpgroup.
constexpr uint32_t kColumns = 512, kColS = 128, kColO = 256;

// Products of parts, small ones first: part x of A times part y of B.
__device__ constexpr int part_a(int x) { return x == 0 ? 2 : x == 2 || x == 3 ? 1 : 0; }
__device__ constexpr int part_b(int x) { return x == 1 ? 2 : x == 2 || x == 4 ? 1 : 0; }

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
// Bounded wait for what was issued, whatever has failed.
__device__ void mbar_drain(uint32_t bar) {
  const unsigned long long t0 = now_ns();
  while (!mbar_try_wait(bar, 0) && now_ns() - t0 < kTimeoutNs) {
  }
}
// Bounded wait; false once any wait of the CTA has run out.
__device__ bool mbar_wait(uint32_t bar, unsigned parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  unsigned spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 63) == 0) {
      if (*failed) return false;
      if (now_ns() - t0 > kTimeoutNs) {
        *failed = 1;
        return false;
      }
    }
  }
  return true;
}

// Operand tiles of 128-byte rows with 128-byte swizzle, 8-row atoms of 1024
// bytes. K-major: a row is 64 entries along K; `lead` is not used. MN-major:
// a row is 64 entries along N at one K; `lead` bytes to the next 64 along N.
__device__ __forceinline__ uint64_t sw128(uint32_t addr, uint32_t lead) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)((lead >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 16 columns of this thread's lane.
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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
// Orders this thread's shared-memory writes before the tensor cores' reads.
__device__ __forceinline__ void fence_operands() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// 2^x; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16x2(float x0, float x1) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(x1), "f"(x0));
  return w;
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
// Two values as N bf16 parts each: x = p[0] + p[1] + ..., each the rounding
// of what the ones before leave.
template <int N>
__device__ __forceinline__ void parts(float x0, float x1, uint32_t* p) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    p[i] = bf16x2(x0, x1);
    x0 -= low(p[i]);
    x1 -= high(p[i]);
  }
}

// Byte of 16-byte group c (8 entries) of row r in a tile of `rows` rows.
__device__ __forceinline__ uint32_t at_sw128(int rows, int r, int c) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_tree_tc(TreeArgs a) {
  using C = Tc<T, HD>;
  constexpr bool kF32 = C::kF32;
  constexpr int kKeys = C::kKeys, kStages = C::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages],
      v_empty[kStages], s_full[2], p_full[2], o_full[2], o_empty[2], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ float2 ml[kRows];  // of the second warpgroup
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (saddr(raw) + 1023u) & ~1023u;
  uint8_t* const gbase = raw + (base - saddr(raw));
  const uint32_t sq = base, skv = base + C::kParts * C::kQPart;
  const uint32_t sraw = skv + kStages * 2 * C::kTile;
  auto k_tile = [&](int s) { return skv + s * 2 * C::kTile; };
  auto v_tile = [&](int s) { return skv + s * 2 * C::kTile + C::kTile; };
  const int split = blockIdx.x, head = blockIdx.y, r0 = blockIdx.z * kRows;
  const int R = a.t * a.group;
  pdl_trigger();
  pdl_wait();
  const int n = tree_cached(a);
  const int tiles = (n + kKeys - 1) / kKeys, per = (tiles + a.splits - 1) / a.splits;
  const int tile0 = split * per, nt = min(tiles, tile0 + per) - tile0;
  if (nt <= 0) return;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) {
      mbar_init(saddr(&k_full[s]), C::kLoaded);
      mbar_init(saddr(&v_full[s]), C::kLoaded);
      mbar_init(saddr(&k_empty[s]), 1);
      mbar_init(saddr(&v_empty[s]), 1);
    }
    for (int w = 0; w < 2; w++) {
      mbar_init(saddr(&s_full[w]), 1);
      mbar_init(saddr(&p_full[w]), 128);
      mbar_init(saddr(&o_full[w]), 1);
      mbar_init(saddr(&o_empty[w]), 128);
    }
    mbar_init(saddr(&done), 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     saddr(&tmem_slot)),
                 "r"(kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  // Queries, zeros for rows behind the last.
  for (int i = threadIdx.x; i < kRows * (HD / 8); i += kThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8), row = r0 + r;
    uint4 w[C::kParts];
#pragma unroll
    for (int p = 0; p < C::kParts; p++) w[p] = make_uint4(0, 0, 0, 0);
    if (row < R) {
      const int tok = row / a.group;
      const T* q = static_cast<const T*>(a.q) + tok * a.ldq +
                   (size_t)(head * a.group + row - tok * a.group) * HD + c * 8;
      if constexpr (kF32) {
        const float4 x = reinterpret_cast<const float4*>(q)[0];
        const float4 y = reinterpret_cast<const float4*>(q)[1];
        uint32_t e[4][3];
        parts<3>(x.x, x.y, e[0]);
        parts<3>(x.z, x.w, e[1]);
        parts<3>(y.x, y.y, e[2]);
        parts<3>(y.z, y.w, e[3]);
#pragma unroll
        for (int p = 0; p < 3; p++) w[p] = make_uint4(e[0][p], e[1][p], e[2][p], e[3][p]);
      } else {
        w[0] = *reinterpret_cast<const uint4*>(q);
      }
    }
#pragma unroll
    for (int p = 0; p < C::kParts; p++)
      *reinterpret_cast<uint4*>(gbase + p * C::kQPart + at_sw128(kRows, r, c)) = w[p];
  }
  fence_operands();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp >= 8) {
    // 384 threads of 168 registers: 2 x 128 x 208 + 128 x 88 make as many.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      if (lane == 0) {
        auto scores = [&](int i) {  // S of tile i
          const int s = i % kStages, w = i & 1;
          if (!mbar_wait(saddr(&k_full[s]), (i / kStages) & 1, &failed)) return false;
          fence_after();
          bool add = false;
#pragma unroll
          for (int x = 0; x < (kF32 ? 6 : 1); x++) {
            const int pq = kF32 ? part_a(x) : 0, pk = kF32 ? part_b(x) : 0;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
              const uint32_t at = (k / 4), in = (k % 4) * 32;
              mma_ss(tmem + w * kColS + C::kS, sw128(sq + pq * C::kQPart + at * kRows * 128 + in, 16),
                     sw128(k_tile(s) + pk * C::kPart + at * kKeys * 128 + in, 16), C::kDescS, add);
              add = true;
            }
          }
          mma_commit(saddr(&s_full[w]));
          mma_commit(saddr(&k_empty[s]));
          return true;
        };
        bool ok = scores(0) && (nt < 2 || scores(1));
        for (int i = 0; ok && i < nt; i++) {
          const int s = i % kStages, w = i & 1, turn = i >> 1;
          ok = mbar_wait(saddr(&p_full[w]), turn & 1, &failed) &&
               mbar_wait(saddr(&v_full[s]), (i / kStages) & 1, &failed) &&
               (turn == 0 || mbar_wait(saddr(&o_empty[w]), (turn - 1) & 1, &failed));
          if (!ok) break;
          fence_after();
          bool add = false;
#pragma unroll
          for (int x = 0; x < (kF32 ? 6 : 2); x++) {
            const int pp = kF32 ? part_a(x) : 1 - x, pv = kF32 ? part_b(x) : 0;
#pragma unroll
            for (int k = 0; k < kKeys / 16; k++) {
              // P's columns: per 32 keys, 16 of each part.
              const uint32_t p = (k / 2) * C::kPParts * 16 + pp * 16 + (k % 2) * 8;
              mma_ts(tmem + kColO + w * 128, tmem + w * kColS + p,
                     sw128(v_tile(s) + pv * C::kPart + k * 2048, kKeys * 128), C::kDescO, add);
              add = true;
            }
          }
          mma_commit(saddr(&o_full[w]));
          mma_commit(saddr(&v_empty[s]));
          // The next scores of this warpgroup overwrite the P that this
          // product reads.
          if (i + 2 < nt)
            ok = mbar_wait(saddr(&o_full[w]), turn & 1, &failed) && scores(i + 2);
        }
        // Nothing issued here outlives the tensor memory.
        mma_commit(saddr(&done));
        mbar_drain(saddr(&done));
      }
      __syncwarp();
    } else {
      const T* kbase = static_cast<const T*>(a.k) + (size_t)head * a.ctx * HD;
      const T* vbase = static_cast<const T*>(a.v) + (size_t)head * a.ctx * HD;
      if constexpr (!kF32) {
        // Each loader warp has one of the three stages: it waits for what it
        // copied without holding up the other stages.
        const int s = warp - 9;
        for (int i = s; i < nt; i += kStages) {
          const unsigned turn = (unsigned)(i / kStages);
          const int row = (tile0 + i) * kKeys, rows = min(kKeys, n - row);
          auto copy = [&](const T* from, uint32_t to) {
#pragma unroll 8
            for (int x = lane; x < kKeys * (HD / 8); x += 32) {
              const int r = x / (HD / 8), c = x % (HD / 8);
              const bool in = r < rows;  // zeros behind the last key
              cp_async16(to + at_sw128(kKeys, r, c),
                         from + (size_t)(in ? row + r : 0) * HD + c * 8, in ? 16 : 0);
            }
            cp_async_commit();
          };
          if (turn && !mbar_wait(saddr(&k_empty[s]), (turn - 1) & 1, &failed)) break;
          copy(kbase, k_tile(s));
          if (turn && !mbar_wait(saddr(&v_empty[s]), (turn - 1) & 1, &failed)) break;
          copy(vbase, v_tile(s));
          cp_async_wait<1>();
          fence_operands();
          mbar_arrive(saddr(&k_full[s]));
          cp_async_wait<0>();
          fence_operands();
          mbar_arrive(saddr(&v_full[s]));
        }
        cp_async_wait<0>();
      } else {
        const int id = threadIdx.x - 288;
        // Units of 32 keys: K, K, V, V of each tile. The next unit's rows
        // stream into the other raw buffer while this one's become parts.
        constexpr int kUnits = kKeys / C::kRawKeys;
        auto fetch = [&](int u) {
          if (u < nt * 2 * kUnits) {
            const int tile = u / (2 * kUnits), half = u % kUnits;
            const bool is_v = u / kUnits & 1;
            const int row = (tile0 + tile) * kKeys + half * C::kRawKeys;
            const int rows = min(C::kRawKeys, n - row);
            const T* from = is_v ? vbase : kbase;
            const uint32_t to = sraw + (u & 1) * (C::kRaw / 2);
#pragma unroll 4
            for (int x = id; x < C::kRawKeys * (HD / 4); x += kLoaders) {
              const int r = x / (HD / 4), c = x % (HD / 4);
              const bool in = r < rows;
              cp_async16(to + x * 16, from + (size_t)(in ? row + r : 0) * HD + c * 4, in ? 16 : 0);
            }
          }
          cp_async_commit();
        };
        fetch(0);
        bool ok = true;
        for (int u = 0; u < nt * 2 * kUnits; u++) {
          const int i = u / (2 * kUnits), half = u % kUnits, s = i % kStages;
          const bool is_v = u / kUnits & 1;
          cp_async_wait<0>();
          // All loaders' copies of this unit have landed, and all are done
          // with the other buffer.
          asm volatile("bar.sync 1, %0;" ::"n"(kLoaders) : "memory");
          fetch(u + 1);
          if (half == 0 && i >= kStages)
            ok = ok && mbar_wait(saddr(is_v ? &v_empty[s] : &k_empty[s]), (i / kStages - 1) & 1,
                                 &failed);
          // (A wait that ran out leaves nothing to do but to stay in step.)
          const uint8_t* from = gbase + (sraw - base) + (u & 1) * (C::kRaw / 2);
          uint8_t* to = gbase + ((is_v ? v_tile(s) : k_tile(s)) - base);
          if (ok) {
#pragma unroll 2
            for (int x = id; x < C::kRawKeys * (HD / 8); x += kLoaders) {
              const int r = x / (HD / 8), c = x % (HD / 8);
              const float4 f = *reinterpret_cast<const float4*>(from + (r * HD + c * 8) * 4);
              const float4 g = *reinterpret_cast<const float4*>(from + (r * HD + c * 8) * 4 + 16);
              uint32_t e[4][3];
              parts<3>(f.x, f.y, e[0]);
              parts<3>(f.z, f.w, e[1]);
              parts<3>(g.x, g.y, e[2]);
              parts<3>(g.z, g.w, e[3]);
              const uint32_t at = at_sw128(kKeys, half * C::kRawKeys + r, c);
#pragma unroll
              for (int p = 0; p < 3; p++)
                *reinterpret_cast<uint4*>(to + p * C::kPart + at) =
                    make_uint4(e[0][p], e[1][p], e[2][p], e[3][p]);
            }
          }
          if (half == kUnits - 1 && ok) {
            fence_operands();
            mbar_arrive(saddr(is_v ? &v_full[s] : &k_full[s]));
          }
        }
        cp_async_wait<0>();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // Softmax: this thread's row is lane 32 (warp % 4) + lane of the tile.
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tp = tmem + w * kColS + lanes, ts = tp + C::kS, to = tmem + kColO + w * 128 + lanes;
    // Scores in units of log2, so that the softmax is exp2.
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    float o[HD], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < HD; i++) o[i] = 0.f;
    for (int i = w; i < nt; i += 2) {
      const int turn = i >> 1;
      const int keys = min(kKeys, n - (tile0 + i) * kKeys);
      if (!mbar_wait(saddr(&s_full[w]), turn & 1, &failed)) break;
      fence_after();
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kKeys / 32; c++) {
        uint32_t s[32];
        tmem_ld(ts + c * 32, s);
        tmem_wait_ld();
        if ((c + 1) * 32 <= keys) {
#pragma unroll
          for (int j = 0; j < 32; j++) top = fmaxf(top, __uint_as_float(s[j]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++)
            if (c * 32 + j < keys) top = fmaxf(top, __uint_as_float(s[j]));
        }
      }
      const float next = fmaxf(m, top * scale);
      const float keep = ex2(m - next);  // 0 before the first key
      const float shift = next == -INFINITY ? 0.f : next;
      m = next;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < kKeys / 32; c++) {
        uint32_t s[32];
        tmem_ld(ts + c * 32, s);
        tmem_wait_ld();
        uint32_t p[C::kPParts][16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x0 = ex2(fmaf(__uint_as_float(s[j]), scale, -shift));
          float x1 = ex2(fmaf(__uint_as_float(s[j + 1]), scale, -shift));
          if ((c + 1) * 32 > keys) {
            if (c * 32 + j >= keys) x0 = 0.f;
            if (c * 32 + j + 1 >= keys) x1 = 0.f;
          }
          sum += x0 + x1;
          uint32_t e[C::kPParts];
          parts<C::kPParts>(x0, x1, e);
#pragma unroll
          for (int y = 0; y < C::kPParts; y++) p[y][j / 2] = e[y];
        }
#pragma unroll
        for (int y = 0; y < C::kPParts; y++) tmem_st16(tp + (c * C::kPParts + y) * 16, p[y]);
      }
      l = l * (m == -INFINITY ? 1.f : keep) + sum;
      tmem_wait_st();
      fence_before();
      mbar_arrive(saddr(&p_full[w]));
      if (!mbar_wait(saddr(&o_full[w]), turn & 1, &failed)) break;
      fence_after();
#pragma unroll
      for (int c = 0; c < HD / 32; c++) {
        uint32_t x[32];
        tmem_ld(to + c * 32, x);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j++)
          o[c * 32 + j] = fmaf(o[c * 32 + j], m == -INFINITY ? 1.f : keep, __uint_as_float(x[j]));
      }
      fence_before();
      mbar_arrive(saddr(&o_empty[w]));
    }
    // A wait that ran out leaves NaN: no result passes for a complete one.
    if (failed) l = o[0] = __int_as_float(0x7FC00000);
    if (w == 1) ml[r] = make_float2(m, l);
    // Both warpgroups are past their last matrix instruction: the operands'
    // memory is free.
    asm volatile("bar.sync 2, 256;" ::: "memory");
    float* join = reinterpret_cast<float*>(gbase) + r * (HD + 4);
    if (w == 1) {
#pragma unroll
      for (int i = 0; i < HD; i += 4)
        *reinterpret_cast<float4*>(join + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    if (w == 0) {
      const float2 y = ml[r];
      const float both = fmaxf(m, y.x);
      const float f = both == -INFINITY ? 1.f : ex2(m - both);
      const float g = both == -INFINITY ? 1.f : ex2(y.x - both);
#pragma unroll
      for (int i = 0; i < HD; i += 4) {
        float4 v = *reinterpret_cast<float4*>(join + i);
        v.x = fmaf(o[i], f, v.x * g);
        v.y = fmaf(o[i + 1], f, v.y * g);
        v.z = fmaf(o[i + 2], f, v.z * g);
        v.w = fmaf(o[i + 3], f, v.w * g);
        *reinterpret_cast<float4*>(join + i) = v;
      }
      if (r0 + r < R)
        a.ml[((size_t)split * a.kh + head) * R + r0 + r] = make_float2(both, l * f + y.y * g);
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    float* part = a.part + (((size_t)split * a.kh + head) * R + r0) * HD;
    const int rows = min(kRows, R - r0);
    for (int i = threadIdx.x; i < rows * (HD / 4); i += 256) {
      const int rr = i / (HD / 4), c = i % (HD / 4);
      reinterpret_cast<float4*>(part)[i] =
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(gbase) + rr * (HD + 4) + c * 4);
    }
    fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns)
                 : "memory");
  }
}

template <typename T, int HD>
cudaError_t launch_tc(const TreeArgs& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[kDevices];
  constexpr size_t bytes = Tc<T, HD>::kBytes;
  const cudaError_t e = allow_smem(k_tree_tc<T, HD>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  const int rows = a.t * a.group;
  return try_launch(k_tree_tc<T, HD>, dim3(a.splits, a.kh, (rows + kRows - 1) / kRows),
                    dim3(kThreads), bytes, 1, s, a);
}

}  // namespace

int tree_tc_keys(bool f32) { return f32 ? Tc<float, 128>::kKeys : Tc<uint16_t, 128>::kKeys; }

cudaError_t tree_tc(const TreeArgs& a, bool f32, int head_dim, int dev, cudaStream_t s) {
  if (f32) return head_dim == 128 ? launch_tc<float, 128>(a, dev, s) : launch_tc<float, 64>(a, dev, s);
  return head_dim == 128 ? launch_tc<uint16_t, 128>(a, dev, s) : launch_tc<uint16_t, 64>(a, dev, s);
}

}  // namespace sg
