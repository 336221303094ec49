// strasgpt_k_attn_tree, cached keys, for many rows per kv head: tcgen05.
//
// A CTA has 128 rows (drafted token, q head) of one kv head and a share of
// the cached keys, which all of its rows see. Sixteen warps: two warpgroups
// of softmax, one thread per row, that take the key tiles in turn; a warp
// that issues Q K^T and one that issues P V, so that neither waits for what
// the other waits for; six that bring in keys and values. Per tile of 64
// keys: S = Q K^T into tensor memory; its warpgroup reads S, subtracts the
// running maximum and writes P = 2^(S - m) over it, as bf16 parts; then
// O (+)= P V in tensor memory. Each warpgroup has its own maximum, sum and
// output, joined at the end, so that one's softmax runs under the other's
// matrix instructions.
//
// bf16: K and V by TMA, a warp each; Q in shared memory (128 entries) or
// tensor memory (64); O stays in tensor memory. A new maximum rescales it
// only when it is 2^8 above the one that P is relative to (P is at most 2^8
// then), which happens in the first few tiles as a rule.
// fp32: rows by bulk copies into a ring, from which six warps write their
// parts. The tensor cores' sums are cut, not rounded, so each tile's O starts
// from zero and is added, scaled, to the warpgroup's registers.
//
// P, and fp32's Q, are operands in tensor memory: read from shared memory, Q
// alone would take two thirds of its bandwidth at 64 keys a tile. Keys and
// values lie in shared memory as rows of 64 head entries (128 bytes, 128-byte
// swizzle): K-major for Q K^T, the same rows MN-major for P V.
//
// Precision. bf16: operands as they are, P as two bf16 parts (2^-17). fp32:
// every operand as three bf16 parts of 8 bits each, all 24 of them, and the six
// products that matter (the others are below 2^-24).
//
// Measured, 8 kv heads of head_dim 128: 256 rows over 65500 bf16 keys 97 us
// (2.8 TB/s of cache, 710 TFLOP/s), over 32768 fp32 keys 170 us (1.6 TB/s,
// 200 TFLOP/s); 32 rows over 128000 keys 93 us (5.6 TB/s) and 301 us (3.5
// TB/s), in short runs; calls one after another for a second take 115, 198 and
// (bf16) 110 us. What bounds 128 rows and more: bf16, 0.7 us per tile, the
// matrix instructions (0.4 us: 32 cycles per 16 entries of Q K^T from tensor
// memory, 48 from shared memory, 64 per 16 keys and part of P V) and the
// hand-overs between them and the softmax; fp32, 2.9 us per tile, the six warps that make
// parts (0.9 us for 64 rows, and as much again in waiting and handing over),
// while the matrix instructions take 1.6. Two fp16 parts of scaled rows and
// half the matrix instructions were slower (226 us): the rows' largest values
// cost those warps more than the third part.
#include "attn_tree.h"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <type_traits>

namespace sg {
namespace {

constexpr int kRows = kTreeTcRows;
constexpr int kThreads = 512;
constexpr int kKeys = 64;        // of a tile
constexpr int kLoadWarps = 6;
constexpr int kLoaders = 32 * kLoadWarps;
constexpr unsigned long long kTimeoutNs = 2000000000ULL;

template <typename T, int HD>
struct Tc {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kParts = kF32 ? 3 : 1;           // of q, k, v
  static constexpr int kPParts = kF32 ? 3 : 2;          // of the probabilities
  static constexpr int kPart = kKeys * HD * 2;          // bytes of a tile's part
  static constexpr int kTile = kParts * kPart;          // of K, or of V
  // bf16: stages filled by TMA. fp32: one, and rows on their way to parts in
  // a ring of units, a tile's keys or values.
  static constexpr int kStages = kF32 ? 1 : HD == 128 ? 6 : 8;
  static constexpr int kLoaded = kF32 ? kLoaders : 1;  // arrivals per filled tile
  static constexpr int kUnit = kKeys * HD * 4;
  static constexpr int kRing = kF32 ? 4 : 0;
  static constexpr int kJoin = kRows * (HD + 4) * 4;    // the warpgroups' join
  // Where Q has no room in tensor memory beside four regions of scores (bf16,
  // 128 entries) it lies in shared memory.
  static constexpr bool kQShared = !kF32 && HD == 128;
  static constexpr int kQ = kQShared ? kRows * HD * 2 : 0;
  static constexpr int kOperands = kStages * 2 * kTile + kRing * kUnit + kQ;
  static constexpr int kUsed = (kOperands > kJoin ? kOperands : kJoin) + 1024;
  // At least half of an SM's: the CTA has all of the SM's tensor memory.
  static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  // Tensor memory columns: Q; regions of S and then P (in an fp32 region S
  // starts at column 32: P's parts of 16 keys, which overwrite it from the
  // start, reach no scores that are still to be read); O.
  static constexpr int kSBuffers = kF32 ? 2 : 4, kOBuffers = kF32 ? 1 : 2;
  static constexpr uint32_t kRegion = kF32 ? 96 : 64, kS = kF32 ? 32 : 0;
  static constexpr uint32_t kColS = kQShared ? 0 : kParts * HD / 2;
  static constexpr uint32_t kColO = kColS + kSBuffers * kRegion;
  static_assert(kColO + kOBuffers * HD <= 512, "tensor memory has 512 columns");
  // Instruction descriptors: fp32 sums of bf16, M = 128; S: N = keys, K
  // K-major; O: N = head entries, V MN-major.
  static constexpr uint32_t kBase =
      (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t kDescS = kBase | ((uint32_t)(kKeys >> 3) << 17);
  static constexpr uint32_t kDescO = kBase | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
};
constexpr uint32_t kColumns = 512;

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
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// 64 head entries (x a multiple of 64: 128 bytes) of 64 cache rows from `row`
// on into a tile's panel.
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int row,
                                         int head, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(bar)
      : "memory");
}
// `bytes` (a multiple of 16) as they are; both addresses 16-byte aligned.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst), "l"(src), "r"(bytes), "r"(bar)
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
// Bounded wait for what was issued, whatever has failed.
__device__ __forceinline__ void mbar_drain(uint32_t bar, unsigned parity) {
  const unsigned long long t0 = now_ns();
  while (!mbar_try_wait(bar, parity) && now_ns() - t0 < kTimeoutNs) {
  }
}
// Bounded wait; false once any wait of the CTA has run out.
__device__ bool mbar_wait(uint32_t bar, unsigned parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*failed) return false;
    if (now_ns() - t0 > kTimeoutNs) {
      *failed = 1;
      return false;
    }
  }
  return true;
}

// The same for a whole warp, which stays together: the tensor-memory and
// barrier instructions that follow are for converged warps.
__device__ __forceinline__ bool warp_wait(uint32_t bar, unsigned parity, volatile int* failed) {
  const bool ok = mbar_wait(bar, parity, failed);
  return __all_sync(0xFFFFFFFFu, ok);
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
// One thread of a converged warp. The matrix instructions are issued under
// its predicate and not inside a branch, so that their operands, the same in
// all threads, can stay in uniform registers: a branch took 100 cycles per
// instruction.
__device__ __forceinline__ uint32_t elect() {
  uint32_t one;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(one));
  return one;
}
// D (+)= A B, A in shared memory; in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add, uint32_t issue) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool add, uint32_t issue) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(issue)
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
// 16 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// Until the loads issued have arrived; r is what one of them fills (no use of
// it may move ahead of the wait).
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  tmem_ld16(addr, r);
  tmem_ld16(addr + 16, r + 16);
}
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
  tmem_wait_ld(r);
  tmem_wait_ld(r + 16);
}
// 16, 8 columns of this thread's lane.
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
// The upper halves of two words: two values cut to bf16.
__device__ __forceinline__ uint32_t upper(float x0, float x1) {
  return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}
__device__ __forceinline__ float rest(float x) {  // what the cut leaves, exact
  return x - __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}
// Two values as bf16 parts, x = p[0] + p[1] + ...: N = 3 cuts 8 bits off each
// time and loses nothing; N = 2 rounds the second part.
template <int N>
__device__ __forceinline__ void parts(float x0, float x1, uint32_t* p) {
  p[0] = upper(x0, x1);
  x0 = rest(x0);
  x1 = rest(x1);
  if constexpr (N == 2) {
    p[1] = bf16x2(x0, x1);
  } else {
    p[1] = upper(x0, x1);
    p[2] = upper(rest(x0), rest(x1));
  }
}

// Two fp32 operations in one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack(float x, float y) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ void unpack(f32x2 v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// What cutting both values to bf16 leaves.
__device__ __forceinline__ f32x2 rest2(f32x2 v) {
  float x, y;
  unpack(v, x, y);
  const f32x2 cut = pack(__uint_as_float(__float_as_uint(x) & 0xFFFF0000u),
                         __uint_as_float(__float_as_uint(y) & 0xFFFF0000u));
  return fma2(cut, pack(-1.f, -1.f), v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// Byte of 16-byte group c (8 entries) of row r in a tile of `rows` rows.
__device__ __forceinline__ uint32_t at_sw128(int rows, int r, int c) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    k_tree_tc(TreeArgs a, const __grid_constant__ CUtensorMap k_map,
              const __grid_constant__ CUtensorMap v_map) {
  using C = Tc<T, HD>;
  constexpr bool kF32 = C::kF32;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages],
      v_empty[kStages], s_full[C::kSBuffers], p_full[C::kSBuffers], s_empty[C::kSBuffers],
      o_full[2], o_empty[2], raw_full[C::kRing ? C::kRing : 1],
      raw_empty[C::kRing ? C::kRing : 1], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ float2 ml[kRows];  // of the second warpgroup
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (saddr(raw) + 1023u) & ~1023u;
  uint8_t* const gbase = raw + (base - saddr(raw));
  auto k_tile = [&](int s) { return base + s * 2 * C::kTile; };
  auto v_tile = [&](int s) { return base + s * 2 * C::kTile + C::kTile; };
  const uint32_t q_at = base + kStages * 2 * C::kTile;
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
    for (int b = 0; b < C::kSBuffers; b++) {
      mbar_init(saddr(&s_full[b]), 1);
      mbar_init(saddr(&p_full[b]), 128);
      mbar_init(saddr(&s_empty[b]), 1);
    }
    for (int w = 0; w < 2; w++) {
      mbar_init(saddr(&o_full[w]), 1);
      mbar_init(saddr(&o_empty[w]), 128);
    }
    for (int x = 0; x < C::kRing; x++) {
      mbar_init(saddr(&raw_full[x]), 1);
      mbar_init(saddr(&raw_empty[x]), kLoaders);
    }
    mbar_init(saddr(&done), 2);
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
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  // 512 threads of 128 registers: 2 x 128 x 208 + 2 x 128 x 48 make as many.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    const uint32_t one = elect();
    if (warp == 8) {
      // S of every tile. Queries are there once the first warpgroup has
      // written them.
      asm volatile("bar.sync 3, 160;" ::: "memory");
      fence_after();
#pragma unroll 1
      for (int i = 0; i < nt; i++) {
        const int s = i % kStages, b = i % C::kSBuffers;
        // The region's last P has been multiplied.
        if (i >= C::kSBuffers &&
            !warp_wait(saddr(&s_empty[b]), (i / C::kSBuffers - 1) & 1, &failed))
          break;
        if (!warp_wait(saddr(&k_full[s]), (i / kStages) & 1, &failed)) break;
        fence_after();
        const uint64_t k0 = sw128(k_tile(s), 16), q0 = sw128(q_at, 16);
        const uint32_t d = tmem + C::kColS + b * C::kRegion + C::kS;
#pragma unroll
        for (int x = 0; x < (kF32 ? 6 : 1); x++) {
          const int pq = kF32 ? part_a(x) : 0, pk = kF32 ? part_b(x) : 0;
#pragma unroll
          for (int k = 0; k < HD / 16; k++) {
            const uint64_t kd = k0 + ((pk * C::kPart + (k / 4) * kKeys * 128 + (k % 4) * 32) >> 4);
            if constexpr (C::kQShared)
              mma_ss(d, q0 + (((k / 4) * kRows * 128 + (k % 4) * 32) >> 4), kd, C::kDescS,
                     x + k > 0, one);
            else
              mma_ts(d, tmem + pq * (HD / 2) + k * 8, kd, C::kDescS, x + k > 0, one);
          }
        }
        mma_commit(saddr(&s_full[b]), one);
        mma_commit(saddr(&k_empty[s]), one);
      }
      // Nothing issued here outlives the tensor memory.
      mma_commit(saddr(&done), one);
      mbar_drain(saddr(&done), 0);
      __syncwarp();
    } else if (warp == 9) {
      // O of every tile.
#pragma unroll 1
      for (int i = 0; i < nt; i++) {
        const int s = i % kStages, b = i % C::kSBuffers, w = i & 1, o = kF32 ? 0 : w;
        // fp32: the last product in these columns has been read. (O's barriers
        // go by warpgroup, so that who waits on one has seen all its phases.)
        const int last = i - 1;
        if (!warp_wait(saddr(&p_full[b]), (i / C::kSBuffers) & 1, &failed) ||
            !warp_wait(saddr(&v_full[s]), (i / kStages) & 1, &failed) ||
            (kF32 && last >= 0 &&
             !warp_wait(saddr(&o_empty[last & 1]), (last >> 1) & 1, &failed)))
          break;
        fence_after();
        const uint64_t v0 = sw128(v_tile(s), kKeys * 128);
        const uint32_t d = tmem + C::kColO + o * HD, p0 = tmem + C::kColS + b * C::kRegion;
#pragma unroll
        for (int x = 0; x < (kF32 ? 6 : 2); x++) {
          const int pp = kF32 ? part_a(x) : 1 - x, pv = kF32 ? part_b(x) : 0;
#pragma unroll
          for (int k = 0; k < kKeys / 16; k++)
            // P's columns: per 32 keys, 16 of each part.
            mma_ts(d, p0 + (k / 2) * C::kPParts * 16 + pp * 16 + (k % 2) * 8,
                   v0 + ((pv * C::kPart + k * 2048) >> 4), C::kDescO,
                   x + k > 0 || (!kF32 && i >= 2), one);
        }
        mma_commit(saddr(&o_full[w]), one);
        mma_commit(saddr(&s_empty[b]), one);
        mma_commit(saddr(&v_empty[s]), one);
      }
      mma_commit(saddr(&done), one);
      mbar_drain(saddr(&done), 0);
      __syncwarp();
    } else {
      const T* kbase = static_cast<const T*>(a.k) + (size_t)head * a.ctx * HD;
      const T* vbase = static_cast<const T*>(a.v) + (size_t)head * a.ctx * HD;
      if constexpr (!kF32) {
        // One warp for the keys, one for the values.
        auto load = [&](const CUtensorMap* map, const T* from, bool is_v, uint64_t* full,
                        uint64_t* empty) {
          int asked = nt;
#pragma unroll 1
          for (int i = 0; i < nt; i++) {
            const int s = i % kStages, row = (tile0 + i) * kKeys, rows = min(kKeys, n - row);
            const uint32_t to = is_v ? v_tile(s) : k_tile(s);
            if (i >= kStages && !warp_wait(saddr(&empty[s]), (i / kStages - 1) & 1, &failed)) {
              asked = i;
              break;
            }
            if (rows == kKeys) {
              if (one) {
                mbar_expect_tx(saddr(&full[s]), C::kPart);
#pragma unroll
                for (int p = 0; p < HD / 64; p++)
                  tma_rows(to + p * kKeys * 128, map, p * 64, row, head, saddr(&full[s]));
              }
            } else {
              // The last tile: rows behind the last cached key are zeros and
              // not what the cache has there.
#pragma unroll 4
              for (int x = lane; x < kKeys * (HD / 8); x += 32) {
                const int r = x / (HD / 8), c = x % (HD / 8);
                const bool in = r < rows;
                cp_async16(to + at_sw128(kKeys, r, c),
                           from + (size_t)(in ? row + r : 0) * HD + c * 8, in ? 16 : 0);
              }
              cp_async_commit();
              cp_async_wait<0>();
              fence_operands();
              __syncwarp();
              if (one) mbar_arrive(saddr(&full[s]));
            }
            __syncwarp();
          }
          // Nothing is on its way when the CTA ends, whatever has failed: the
          // last tile asked for in each stage is waited for (those before it
          // were, before it was asked for), by a lane each: a loop over the
          // stages made 256 rows over 65500 bf16 keys 129 us for 115.
          if (lane < kStages && lane < asked)
            mbar_drain(saddr(&full[lane]), tree_last_parity(asked, lane, kStages));
          __syncwarp();
        };
        if (warp == 10) load(&k_map, kbase, false, k_full, k_empty);
        if (warp == 11) load(&v_map, vbase, true, v_full, v_empty);
      } else {
        // Units in the order of their use: K of tile 0, then K of tile i + 1
        // and V of tile i. The rows of the next kRing stream into the ring
        // while this one's become parts.
        constexpr int kRing = C::kRing;
        const int id = threadIdx.x - 320, units = 2 * nt;
        const uint32_t ring = base + kStages * 2 * C::kTile;
        // Tile of unit u, and whether it is of V.
        auto unit = [&](int u, bool& is_v) {
          is_v = u > 0 && (!(u & 1) || u == units - 1);
          return u == 0 ? 0 : u == units - 1 ? nt - 1 : is_v ? u / 2 - 1 : (u + 1) / 2;
        };
        auto fetch = [&](int u) {
          if (u >= units) return;
          bool is_v;
          const int row = (tile0 + unit(u, is_v)) * kKeys;
          const uint32_t bar = saddr(&raw_full[u % kRing]), bytes = min(kKeys, n - row) * HD * 4;
          mbar_expect_tx(bar, bytes);
          bulk_copy(ring + (u % kRing) * C::kUnit, (is_v ? vbase : kbase) + (size_t)row * HD, bytes,
                    bar);
        };
        if (id == 0)
          for (int u = 0; u < kRing; u++) fetch(u);
        int asked = min(kRing, units);  // the last warp's count
        bool ok = true;
#pragma unroll 1
        for (int u = 0; u < units; u++) {
          bool is_v;
          const int i = unit(u, is_v), rows = min(kKeys, n - (tile0 + i) * kKeys);
          // (A wait that ran out leaves nothing to do but to stay in step.)
          ok = ok && warp_wait(saddr(&raw_full[u % kRing]), (u / kRing) & 1, &failed) &&
               (i == 0 || warp_wait(saddr(is_v ? &v_empty[0] : &k_empty[0]), (i - 1) & 1, &failed));
          if (ok) {
            const uint8_t* from = gbase + (ring - base) + (u % kRing) * C::kUnit;
            uint8_t* to = gbase + (is_v ? C::kTile : 0);
            // A warp takes four rows at a time, eight lanes each: rows r and
            // r + 4 in half a warp, which with the swizzle have all banks.
#pragma unroll 1
            for (int it = warp - 10; it < kKeys / 4; it += kLoadWarps) {
              const int r = (it >> 1) * 8 + (it & 1) * 2 + (lane >> 4) + ((lane >> 3) & 1) * 4;
              float4 v[HD / 32];
#pragma unroll
              for (int j = 0; j < HD / 32; j++)
                v[j] = r < rows ? *reinterpret_cast<const float4*>(from + r * HD * 4 + j * 128 +
                                                                   (lane & 7) * 16)
                                : make_float4(0.f, 0.f, 0.f, 0.f);  // behind the last key
              uint8_t* at = to + r * 128 + (lane & 1) * 8;
#pragma unroll
              for (int j = 0; j < HD / 32; j++) {
                uint8_t* p = at + (j >> 1) * kKeys * 128 +
                             ((((j & 1) * 4 + ((lane & 7) >> 1)) ^ (r & 7)) << 4);
                f32x2 x = pack(v[j].x, v[j].y), y = pack(v[j].z, v[j].w);
#pragma unroll
                for (int q = 0; q < 3; q++) {
                  float x0, x1, y0, y1;
                  unpack(x, x0, x1);
                  unpack(y, y0, y1);
                  *reinterpret_cast<uint2*>(p + q * C::kPart) =
                      make_uint2(upper(x0, x1), upper(y0, y1));
                  if (q < 2) {
                    x = rest2(x);
                    y = rest2(y);
                  }
                }
              }
            }
            fence_operands();
            mbar_arrive(saddr(is_v ? &v_full[0] : &k_full[0]));
          }
          mbar_arrive(saddr(&raw_empty[u % kRing]));
          // The last warp refills the buffer of the unit before, which the
          // others are done with by now as a rule.
          if (warp == 15 && u > 0 && u - 1 + kRing < units) {
            ok = ok && warp_wait(saddr(&raw_empty[(u - 1) % kRing]), ((u - 1) / kRing) & 1,
                                 &failed);
            if (one && ok) fetch(u - 1 + kRing);
            asked += ok;
            __syncwarp();
          }
        }
        // After a failure units may still be on their way: their memory is
        // this CTA's until they have landed. (The last warp has waited for
        // all of them otherwise.)
        if (warp == 15 && !ok && lane < kRing && lane < asked)
          mbar_drain(saddr(&raw_full[lane]), tree_last_parity(asked, lane, kRing));
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // Softmax: this thread's row is lane 32 (warp % 4) + lane of the tile.
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    if (w == 0) {
      // Queries into tensor (or shared) memory, zeros for rows behind the last.
      const int row = r0 + r, tok = row < R ? row / a.group : 0;
      const T* q = static_cast<const T*>(a.q) + tok * a.ldq +
                   (size_t)(head * a.group + (row < R ? row - tok * a.group : 0)) * HD;
      constexpr int kVec = 16 / sizeof(T), kBatch = 8;  // 16-byte loads in flight
#pragma unroll
      for (int c = 0; c < HD / (kVec * kBatch); c++) {
        uint4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; j++) {
          x[j] = reinterpret_cast<const uint4*>(q)[c * kBatch + j];
          if (row >= R) x[j] = make_uint4(0, 0, 0, 0);
        }
        if constexpr (C::kQShared) {
#pragma unroll
          for (int j = 0; j < kBatch; j++)
            *reinterpret_cast<uint4*>(gbase + (q_at - base) + at_sw128(kRows, r, c * kBatch + j)) =
                x[j];
        }
        // 16 entries at a time, 8 columns a part.
#pragma unroll
        for (int h = 0; h < (C::kQShared ? 0 : kBatch * kVec / 16); h++) {
          uint32_t e[C::kParts][8];
          if constexpr (kF32) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const uint4 v = x[4 * h + j];
              uint32_t y[2][3];
              parts<3>(__uint_as_float(v.x), __uint_as_float(v.y), y[0]);
              parts<3>(__uint_as_float(v.z), __uint_as_float(v.w), y[1]);
#pragma unroll
              for (int p = 0; p < 3; p++) {
                e[p][2 * j] = y[0][p];
                e[p][2 * j + 1] = y[1][p];
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint4 v = x[2 * h + j];
              e[0][4 * j] = v.x;
              e[0][4 * j + 1] = v.y;
              e[0][4 * j + 2] = v.z;
              e[0][4 * j + 3] = v.w;
            }
          }
#pragma unroll
          for (int p = 0; p < C::kParts; p++)
            tmem_st8(lanes + p * (HD / 2) + (c * kBatch * kVec / 16 + h) * 8, e[p]);
        }
      }
      if constexpr (C::kQShared) {
        fence_operands();
      } else {
        tmem_wait_st();
        fence_before();
      }
      asm volatile("bar.arrive 3, 160;" ::: "memory");
    }
    // Scores in units of log2, so that the softmax is exp2.
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    float o[kF32 ? HD : 1], m = -INFINITY, l = 0.f;
    const uint32_t to = lanes + C::kColO + (kF32 ? 0 : w * HD);
#pragma unroll
    for (int i = 0; i < (kF32 ? HD : 1); i++) o[i] = 0.f;
    bool ok = true;
#pragma unroll 1
    for (int i = w; i < nt; i += 2) {
      const int b = i % C::kSBuffers;
      const uint32_t tp = lanes + C::kColS + b * C::kRegion, ts = tp + C::kS;
      const int keys = min(kKeys, n - (tile0 + i) * kKeys);
      ok = warp_wait(saddr(&s_full[b]), (i / C::kSBuffers) & 1, &failed);
      if (!ok) break;
      fence_after();
      float keep = 1.f;
      // Partial maxima and sums: short chains.
      float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      f32x2 sum2[2] = {0, 0};
      // P of 32 keys: this thread's scores -> its columns of the region.
      // `all`: none of the tile's keys is behind the last.
      auto probabilities = [&](const uint32_t* s, int c, float shift, auto all) {
        uint32_t p[C::kPParts][16];
        const f32x2 scale2 = pack(scale, scale), shift2 = pack(-shift, -shift);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x0, x1;
          unpack(fma2(pack(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), scale2, shift2), x0,
                 x1);
          x0 = ex2(x0);
          x1 = ex2(x1);
          if constexpr (!decltype(all)::value) {
            if (c * 32 + j >= keys) x0 = 0.f;
            if (c * 32 + j + 1 >= keys) x1 = 0.f;
          }
          f32x2 x = pack(x0, x1);
          sum2[j / 2 % 2] = add2(sum2[j / 2 % 2], x);
          // The parts as in parts<N>().
#pragma unroll
          for (int y = 0; y < C::kPParts; y++) {
            unpack(x, x0, x1);
            p[y][j / 2] = C::kPParts == 2 && y == 1 ? bf16x2(x0, x1) : upper(x0, x1);
            if (y + 1 < C::kPParts) x = rest2(x);
          }
        }
#pragma unroll
        for (int y = 0; y < C::kPParts; y++)
          tmem_st16(tp + (c * C::kPParts + y) * 16, p[y]);
      };
      auto largest = [&](const uint32_t* s, int c, auto all) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x = __uint_as_float(s[j]), y = __uint_as_float(s[j + 1]);
          if constexpr (!decltype(all)::value) {
            if (c * 32 + j >= keys) x = -INFINITY;
            if (c * 32 + j + 1 >= keys) y = -INFINITY;
          }
          top4[j / 2 % 4] = max3(top4[j / 2 % 4], x, y);
        }
      };
      const std::true_type full;
      const std::false_type part;
      const bool whole = keys == kKeys;
      if constexpr (!kF32) {
        uint32_t s[2][32];
        tmem_ld32(ts, s[0]);
        tmem_ld32(ts + 32, s[1]);
        tmem_wait_ld32(s[0]);
        tmem_wait_ld32(s[1]);
        if (whole) {
          largest(s[0], 0, full);
          largest(s[1], 1, full);
        } else {
          largest(s[0], 0, part);
          largest(s[1], 1, part);
        }
        const float next = fmaxf(m, fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * scale);
        if (__any_sync(0xFFFFFFFFu, next > m + 8.f)) {
          // m is what P and O are relative to. (The wait is for the last
          // tile's product; this tile's scores say that the one before is
          // complete, so the parity is not an older phase's.)
          const float f = next == -INFINITY ? 1.f : ex2(m - next);
          m = next;
          l *= f;
          if (i >= 2) {
            ok = warp_wait(saddr(&o_full[w]), ((i - 2) >> 1) & 1, &failed);
            if (!ok) break;
            fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 16; c++) {
              uint32_t x[16];
              tmem_ld16(to + c * 16, x);
              tmem_wait_ld(x);
#pragma unroll
              for (int j = 0; j < 16; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
              tmem_st16(to + c * 16, x);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.f : m;
        if (whole) {
          probabilities(s[0], 0, shift, full);
          probabilities(s[1], 1, shift, full);
        } else {
          probabilities(s[0], 0, shift, part);
          probabilities(s[1], 1, shift, part);
        }
      } else {
        // The scores are read twice: with O in registers there is no room to
        // keep them.
        uint32_t s[32];
        auto tile = [&](auto all) {
          tmem_ld32(ts, s);
          tmem_wait_ld32(s);
          largest(s, 0, all);
          tmem_ld32(ts + 32, s);
          tmem_wait_ld32(s);
          largest(s, 1, all);
          const float next = fmaxf(m, fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * scale);
          keep = next == -INFINITY ? 1.f : ex2(m - next);  // 0 before the first key
          m = next;
          const float shift = next == -INFINITY ? 0.f : next;
          tmem_ld32(ts, s);
          tmem_wait_ld32(s);
          probabilities(s, 0, shift, all);
          tmem_ld32(ts + 32, s);
          tmem_wait_ld32(s);
          probabilities(s, 1, shift, all);
        };
        if (whole)
          tile(full);
        else
          tile(part);
      }
      float even, odd;
      unpack(add2(sum2[0], sum2[1]), even, odd);
      l = l * keep + (even + odd);
      tmem_wait_st();
      fence_before();
      mbar_arrive(saddr(&p_full[b]));
      if constexpr (kF32) {
        ok = warp_wait(saddr(&o_full[w]), (i >> 1) & 1, &failed);
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
          uint32_t x[32];
          tmem_ld32(to + c * 32, x);
          tmem_wait_ld32(x);
#pragma unroll
          for (int j = 0; j < 32; j++)
            o[c * 32 + j] = fmaf(o[c * 32 + j], keep, __uint_as_float(x[j]));
        }
        fence_before();
        mbar_arrive(saddr(&o_empty[w]));
      }
    }
    const bool any = nt > w;  // this warpgroup had a tile
    if constexpr (!kF32) {
      // The last product of this warpgroup, behind the one before (whose
      // older phase has the last one's parity).
      const int turn = (nt - 1 - w) >> 1;
      if (ok && any && turn > 0) ok = warp_wait(saddr(&o_full[w]), (turn - 1) & 1, &failed);
      if (ok && any) ok = warp_wait(saddr(&o_full[w]), turn & 1, &failed);
      fence_after();
    }
    // A wait that ran out leaves NaN: no result passes for a complete one.
    if (failed || !ok) l = __int_as_float(0x7FC00000);
    // 32 outputs of this thread's row.
    auto outputs = [&](int c, float* x) {
      if constexpr (kF32) {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = o[c * 32 + j];
      } else {
        uint32_t y[32];
        tmem_ld32(to + c * 32, y);
        tmem_wait_ld32(y);
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = __uint_as_float(y[j]);
      }
    };
    float* join = reinterpret_cast<float*>(gbase) + r * (HD + 4);
    if (nt > 1) {
      if (w == 1) ml[r] = make_float2(m, l);
      // Both warpgroups are past their last matrix instruction: the operands'
      // memory is free.
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (w == 1) {
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
          float x[32];
          outputs(c, x);
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(join + c * 32 + j) =
                make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        }
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
    }
    if (w == 0) {
      const float2 y = nt > 1 ? ml[r] : make_float2(-INFINITY, 0.f);
      const float both = fmaxf(m, y.x);
      const float f = both == -INFINITY ? 1.f : ex2(m - both);
      const float g = both == -INFINITY ? 1.f : ex2(y.x - both);
      const size_t at = ((size_t)split * a.kh + head) * R + r0 + r;
      if (r0 + r < R) a.ml[at] = make_float2(both, l * f + y.y * g);
#pragma unroll
      for (int c = 0; c < HD / 32; c++) {
        float x[32];
        outputs(c, x);
        float4* part = reinterpret_cast<float4*>(a.part + at * HD + c * 32);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          float4 v = make_float4(x[j] * f, x[j + 1] * f, x[j + 2] * f, x[j + 3] * f);
          if (nt > 1) {
            const float4 z = *reinterpret_cast<const float4*>(join + c * 32 + j);
            v.x = fmaf(z.x, g, v.x);
            v.y = fmaf(z.y, g, v.y);
            v.z = fmaf(z.z, g, v.z);
            v.w = fmaf(z.w, g, v.w);
          }
          if (r0 + r < R) part[j / 4] = v;
        }
      }
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

// Map of a bf16 cache [kh][ctx][hd]: boxes of 64 entries of 64 rows.
cudaError_t cache_map(CUtensorMap* map, const void* base, int kh, int ctx, int hd) {
  const auto encode = encode_fn();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)ctx, (cuuint64_t)kh};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ctx * hd * 2};
  const cuuint32_t box[3] = {64, kKeys, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
                            strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int HD>
cudaError_t launch_tc(const TreeArgs& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[kDevices];
  constexpr size_t bytes = Tc<T, HD>::kBytes;
  cudaError_t e = allow_smem(k_tree_tc<T, HD>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  CUtensorMap k = {}, v = {};
  if (!Tc<T, HD>::kF32) {
    if ((e = cache_map(&k, a.k, a.kh, a.ctx, HD)) != cudaSuccess) return e;
    if ((e = cache_map(&v, a.v, a.kh, a.ctx, HD)) != cudaSuccess) return e;
  }
  const int rows = a.t * a.group;
  return try_launch(k_tree_tc<T, HD>, dim3(a.splits, a.kh, (rows + kRows - 1) / kRows),
                    dim3(kThreads), bytes, 1, s, a, k, v);
}

}  // namespace

int tree_tc_keys() { return kKeys; }

cudaError_t tree_tc(const TreeArgs& a, bool f32, int head_dim, int dev, cudaStream_t s) {
  if (f32) return head_dim == 128 ? launch_tc<float, 128>(a, dev, s) : launch_tc<float, 64>(a, dev, s);
  return head_dim == 128 ? launch_tc<uint16_t, 128>(a, dev, s) : launch_tc<uint16_t, 64>(a, dev, s);
}

}  // namespace sg
