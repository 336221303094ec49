// strasgpt_k_attn_tree: GQA attention of a tree of drafted tokens over the
// cache that ends with the tree's own rows; strasgpt_k_attn_shared: of a batch
// of requests over a prefix that all share and over caches of their own.
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
// (see on_tc). Short caches are latency: 7.0 us for one token over 613 keys,
// both kernels.
//
// Behind a shared prefix: the prefix is read once for all requests' rows, by the
// kernels above (on_tc's from 16 rows a kv head on); the requests' own keys, tiles of
// rows by tiles of keys, are shared out evenly over as many CTAs as the GPU holds,
// which start as the prefix's leave room; k_join adds up both. Measured, captured calls
// in short runs (from Python one after another the longest take some 13 % more), 8 kv heads:
// 64 requests of four heads of 128 bf16 entries, up to 1021 rows each behind 32768,
// 90 us (prefix 47, own rows 41, alone: 4.9 TB/s; join 10); 48 in fp32, 700 behind
// 8191, 107 us (50, 58, 7); 31 requests with up to six drafted tokens of eight heads of
// 64 bf16 entries, 2000 behind 16001, 117 us (66, 57, 9); 16 prompts of up to 96
// tokens behind 8192 rows 205 us (172, 32, 21); two requests behind 613 rows 10 us.
#include "attn_tree.h"

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

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

// Two fp32 operations in one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 x;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x.x), "=f"(x.y) : "l"(v));
  return x;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
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

// A CTA's tokens: of the tree, or of one request.
struct Rows {
  int token0, t;        // first token and tokens
  int r0;               // first row of the CTA, of t * group
  int cached, drafted;  // keys that all rows see, and those behind them
  int late;             // request: token i sees its drafted keys 0..i - late

  __device__ Rows() {}
  __device__ Rows(const TreeArgs& a, int tile_rows) {
    token0 = 0;
    t = a.t;
    r0 = blockIdx.z * tile_rows;
    cached = sg::tree_cached(a);
    drafted = a.drafted;
    late = 0;
  }
  // Whatever stands in device memory, tokens and cache rows are among those
  // that the call names.
  __device__ Rows(const sg::BatchArgs& a, int request, int first_row) {
    r0 = first_row;
    sg::cut_tokens(a.first ? a.first[request] : (long long)request * a.most,
                   a.first ? a.first[request + 1] : (request + 1ll) * a.most, a.t, a.most, &token0,
                   &t);
    const int n = min(max(a.rows[request], 0), a.ctx);
    cached = max(n - t, 0);
    drafted = n - cached;
    late = t - drafted;
  }
};

// Which of the 64 drafted keys from j0 (a multiple of 8, below a word's end)
// token i sees, as bits.
__device__ __forceinline__ u64 seen_of(const TreeArgs& a, const Rows&, int i, int j0) {
  return a.mask[(size_t)i * a.words + (j0 >> 6)] >> (j0 & 63);
}
__device__ __forceinline__ u64 seen_of(const sg::BatchArgs&, const Rows& r, int i, int j0) {
  const int count = i - r.late - j0 + 1;
  return count >= 64 ? ~0ull : count > 0 ? (1ull << count) - 1 : 0;
}
// `rows` cache rows from `row` on to a stage, zeros behind them.
template <typename T, int HD, int THREADS>
__device__ __forceinline__ void load_tile(const T* k, const T* v, int row, int rows, uint32_t ks) {
  using L = Tile<T, HD, THREADS / 32>;
  const uint32_t vs = ks + L::kKeys * L::kKRow;
  constexpr int kVecs = HD * (int)sizeof(T) / 16;
  if (rows == L::kKeys && THREADS % kVecs == 0) {
    // A thread's accesses are a fixed distance apart.
    constexpr int kStep = THREADS / kVecs < 1 ? 1 : THREADS / kVecs;
    const int r = threadIdx.x / kVecs, x = threadIdx.x % kVecs;
    const size_t at = (size_t)(row + r) * HD + x * (16 / sizeof(T));
    const T *from_k = k + at, *from_v = v + at;
    const uint32_t to_k = ks + r * L::kKRow + x * 16, to_v = vs + r * L::kVRow + x * 16;
#pragma unroll
    for (int i = 0; i < L::kKeys; i += kStep) {
      cp_async16(to_k + i * L::kKRow, from_k + (size_t)i * HD, 16);
      cp_async16(to_v + i * L::kVRow, from_v + (size_t)i * HD, 16);
    }
    return;
  }
#pragma unroll 4
  for (int i = threadIdx.x; i < L::kKeys * kVecs; i += THREADS) {
    const int r = i / kVecs, x = i % kVecs;
    const int bytes = r < rows ? 16 : 0;
    const size_t at = (size_t)(row + (r < rows ? r : 0)) * HD + x * (16 / sizeof(T));
    cp_async16(ks + r * L::kKRow + x * 16, k + at, bytes);
    cp_async16(vs + r * L::kVRow + x * 16, v + at, bytes);
  }
}

// The tiles of a split: the cached keys, then the drafted ones. A tile holds
// keys of one kind, never of both.
template <typename T, int HD, int THREADS, int ROWS>
struct Walk {
  using L = Tile<T, HD, THREADS / 32>;
  const T *k, *v;                // of the kv head
  Rows r;
  int n, old_tiles, tile0, tile1;
  uint32_t smem;

  // (The cache's length is read on the device: a captured call serves every
  // later length.)
  __device__ Walk(const TreeArgs& a, const void* stages) : r(a, ROWS) {
    n = r.cached;
    old_tiles = (n + L::kKeys - 1) / L::kKeys;
    const int tiles = old_tiles + (r.drafted + L::kKeys - 1) / L::kKeys;
    const int per = (tiles + a.splits - 1) / a.splits;
    tile0 = blockIdx.x * per;
    tile1 = min(tiles, tile0 + per);
    k = static_cast<const T*>(a.k) + (size_t)blockIdx.y * a.ctx * HD;
    v = static_cast<const T*>(a.v) + (size_t)blockIdx.y * a.ctx * HD;
    smem = saddr(stages);
  }
  __device__ int count() const { return max(0, tile1 - tile0); }
  __device__ const Rows& rows(int) const { return r; }
  __device__ int head(int) const { return blockIdx.y; }
  // Tile i of the split: first cache row and rows.
  __device__ void extent(int i, int& row, int& rows) const {
    const int tile = tile0 + i;
    const bool old = tile < old_tiles;
    const int k0 = (old ? tile : tile - old_tiles) * L::kKeys;
    row = old ? k0 : n + k0;
    rows = min(L::kKeys, (old ? n : r.drafted) - k0);
  }
  // Its rows, and its first key's drafted index, negative if it holds cached ones.
  __device__ void keys(int i, int& rows, int& j0) const {
    int row;
    extent(i, row, rows);
    j0 = tile0 + i < old_tiles ? -1 : row - n;
  }
  __device__ bool last(int i) const { return tile0 + i + 1 >= tile1; }
  __device__ void fetch(int i) const {
    if (tile0 + i < tile1) {
      int row, rows;
      extent(i, row, rows);
      load_tile<T, HD, THREADS>(k, v, row, rows, smem + i % kStages * L::kStage);
    }
    cp_async_commit();
  }
  __device__ int parts(int) const { return 0; }
  // Where the part of row r (of t * group) lies.
  __device__ size_t part(const TreeArgs& a, const Rows&, int head, int, int r) const {
    return ((size_t)blockIdx.x * a.kh + head) * a.t * a.group + r;
  }
};

// A batch: the tiles of all requests, kv heads and row tiles, in this order, are
// shared out evenly, a run to each CTA, whose fetches go on from one (request, head,
// row tile) to the next. Each of these has a tile at least, which may be empty, if
// there are rows.
//
// Its parts: that of the run with its first tile lies with its rows, those of the
// runs that go on with it lie by CTA; which they are is noted for each row.
//
// One thread looks ahead and notes what the others need of a tile.
template <typename T, int HD, int THREADS, int ROWS>
struct Stream {
  using L = Tile<T, HD, THREADS / 32>;
  struct Note {
    size_t base;       // entries before the cache of the tile's request and head
    int row, rows;     // first cache row, rows
    int j0;            // first key's drafted index, or -1
    int head, token0, t, r0, late;
    int parts;         // runs over the (request, head, row tile); 0: not its first tile
    int last;          // of it, or of this CTA's
  };
  static constexpr int kNotes = 4;  // two tiles ahead, and one that is written
  struct Shared {
    Note notes[kNotes];
    Rows r;
    int request, head, z, tile, tiles, old_tiles;
    long long at, per, end;  // the next tile's number; a CTA's tiles; the last's number + 1
    long long sums[THREADS / 32];
  };
  const sg::BatchArgs& a;
  Shared& s;
  uint32_t smem;
  int tiles_;

  static __device__ int key_tiles(const Rows& r) {
    return max(1, (r.cached + L::kKeys - 1) / L::kKeys + (r.drafted + L::kKeys - 1) / L::kKeys);
  }
  static __device__ int row_tiles(const sg::BatchArgs& a, const Rows& r) {
    return (r.t * a.group + ROWS - 1) / ROWS;
  }
  __device__ void enter(int request) {
    s.request = request;
    s.r = Rows(a, request, 0);
    s.old_tiles = (s.r.cached + L::kKeys - 1) / L::kKeys;
    s.tiles = key_tiles(s.r);
  }
  // Notes the next tile, as this CTA's i-th.
  __device__ void look_ahead(int i) {
    if (s.at >= s.end) return;
    Note& n = s.notes[i % kNotes];
    const bool old = s.tile < s.old_tiles;
    const int k0 = (old ? s.tile : s.tile - s.old_tiles) * L::kKeys;
    n.base = (size_t)s.request * a.stride + (size_t)s.head * a.ctx * HD;
    n.row = old ? k0 : s.r.cached + k0;
    n.rows = max(0, min(L::kKeys, (old ? s.r.cached : s.r.drafted) - k0));
    n.j0 = old ? -1 : k0;
    n.head = s.head;
    n.token0 = s.r.token0;
    n.t = s.r.t;
    n.r0 = s.z * ROWS;
    n.late = s.r.late;
    n.parts = s.tile ? 0 : (int)((s.at + s.tiles - 1) / s.per - blockIdx.x + 1);
    s.at++;
    s.tile++;
    n.last = s.tile == s.tiles || s.at == s.end;
    if (s.tile < s.tiles || s.at == s.end) return;
    s.tile = 0;
    if (++s.z < row_tiles(a, s.r)) return;
    s.z = 0;
    if (++s.head < a.kh) return;
    s.head = 0;
    // (There is one: there are tiles left.)
    do enter(s.request + 1);
    while (s.r.t == 0);
  }

  __device__ Stream(const sg::BatchArgs& args, Shared& shared, const void* stages)
      : a(args), s(shared) {
    smem = saddr(stages);
    // Every thread counts the tiles of some requests in a row; the one that has
    // this CTA's first tile's finds it.
    const int each = (a.requests + THREADS - 1) / THREADS, lane = threadIdx.x & 31;
    const int from = threadIdx.x * each, to = min(a.requests, from + each);
    auto tiles_of = [&](int request) {
      const Rows r(a, request, 0);
      return (long long)key_tiles(r) * row_tiles(a, r) * a.kh;
    };
    long long mine = 0;
    for (int r = from; r < to; r++) mine += tiles_of(r);
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.sums[threadIdx.x >> 5] = upto;
    __syncthreads();
    long long before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
      if (w < (int)(threadIdx.x >> 5)) before += s.sums[w];
      all += s.sums[w];
    }
    const long long per = max(1ll, (all + gridDim.x - 1) / gridDim.x), at = per * blockIdx.x;
    tiles_ = (int)max(0ll, min(per, all - at));
    if (tiles_ && at >= before && at < before + mine) {
      long long left = at - before;
      int r = from;
      for (long long n; left >= (n = tiles_of(r)); r++) left -= n;
      enter(r);
      const int rows = row_tiles(a, s.r);
      s.tile = (int)(left % s.tiles);
      left /= s.tiles;
      s.z = (int)(left % rows);
      s.head = (int)(left / rows);
      s.at = at;
      s.per = per;
      s.end = at + tiles_;
      for (int i = 0; i < kNotes - 1; i++) look_ahead(i);
    }
    __syncthreads();
  }
  __device__ int count() const { return tiles_; }
  __device__ Rows rows(int i) const {
    const Note& n = s.notes[i % kNotes];
    Rows r;
    r.token0 = n.token0;
    r.t = n.t;
    r.r0 = n.r0;
    r.late = n.late;
    return r;
  }
  __device__ int head(int i) const { return s.notes[i % kNotes].head; }
  __device__ void keys(int i, int& rows, int& j0) const {
    rows = s.notes[i % kNotes].rows;
    j0 = s.notes[i % kNotes].j0;
  }
  __device__ bool last(int i) const { return s.notes[i % kNotes].last; }
  // Asks for tile i, if there is one (it is noted). Between two calls is a barrier.
  __device__ void fetch(int i) {
    if (i < tiles_) {
      const Note& n = s.notes[i % kNotes];
      load_tile<T, HD, THREADS>(static_cast<const T*>(a.k) + n.base,
                                static_cast<const T*>(a.v) + n.base, n.row, n.rows,
                                smem + i % kStages * L::kStage);
      if (i >= kStages - 1 && threadIdx.x == 0) look_ahead(i + 1);
    }
    cp_async_commit();
  }
  __device__ int parts(int i) const { return s.notes[i % kNotes].parts; }
  // Where the part of row r of these lies; the first run notes who goes on.
  __device__ size_t part(const sg::BatchArgs& a, const Rows& rows, int head, int parts,
                         int r) const {
    const size_t all = (size_t)a.t * a.group, row = head * all + (size_t)rows.token0 * a.group + r;
    if (!parts) return (a.split0 + 1) * a.kh * all + (size_t)blockIdx.x * ROWS + (r - rows.r0);
    a.where[row] = make_int2(blockIdx.x, parts * 128 + r - rows.r0);
    return a.split0 * a.kh * all + row;
  }
};

// MW warps side by side in rows (16 each), KW in keys.
template <typename T, int HD, int THREADS, int ROWS, typename Args>
using Walker = std::conditional_t<std::is_same<Args, sg::BatchArgs>::value,
                                  Stream<T, HD, THREADS, ROWS>, Walk<T, HD, THREADS, ROWS>>;

template <typename T, int HD, int MW, int KW, typename Args>
__global__ void __launch_bounds__(32 * MW * KW, MW* KW <= 4 ? 2 : 1) k_tree(Args a) {
  using L = Tile<T, HD, MW * KW>;
  constexpr bool kF32 = L::kF32, kBatch = std::is_same<Args, sg::BatchArgs>::value;
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
  // A batch's own tiles follow its prefix's, which they do not need: they start as
  // that one's CTAs leave room. It lets them once all before it is complete, and is
  // waited for at the end: this kernel is complete when both are.
  if constexpr (!kBatch) sg::pdl_wait();
  sg::pdl_trigger();

  using W = Walker<T, HD, kThreads, kRows, Args>;
  auto start = [&] {
    if constexpr (kBatch) {
      __shared__ typename W::Shared shared;
      return W(a, shared, smem);
    } else {
      return W(a, smem);
    }
  };
  W walk = start();
  if (walk.count() == 0) {
    if constexpr (kBatch) sg::pdl_wait();
    return;
  }
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) walk.fetch(s);

  int at = 0;  // tiles gone through
  do {
    const Rows rows_of = walk.rows(at);
    const int head = walk.head(at), R = rows_of.t * a.group, r0 = rows_of.r0;
    const int parts = walk.parts(at);
    // This lane's rows g8 and g8 + 8 of the warp's 16.
    const int rA = r0 + 16 * mw + g8, rB = rA + 8;
    const int tA = rA / a.group, tB = rB / a.group;
    const bool inA = rA < R, inB = rB < R;
    const T* qA = static_cast<const T*>(a.q) + (rows_of.token0 + (inA ? tA : 0)) * a.ldq +
                  (size_t)(head * a.group + (inA ? rA - tA * a.group : 0)) * HD;
    const T* qB = static_cast<const T*>(a.q) + (rows_of.token0 + (inB ? tB : 0)) * a.ldq +
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

    for (bool more = true; more; at++) {
      cp_async_wait<kStages - 2>();
      __syncthreads();
      walk.fetch(at + kStages - 1);  // into the buffer that the last tile left
      int rows, first;
      walk.keys(at, rows, first);
      more = !walk.last(at);
      const bool old = first < 0;
      const unsigned char* ks = smem + at % kStages * L::kStage;
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
          const int j0 = first + k0;  // drafted index, a multiple of 8
          const u64 wA = inA ? seen_of(a, rows_of, tA, j0) : 0;
          const u64 wB = inB ? seen_of(a, rows_of, tB, j0) : 0;
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
    if constexpr (!kBatch) cp_async_wait<0>();
    lA += __shfl_xor_sync(0xFFFFFFFFu, lA, 1);
    lA += __shfl_xor_sync(0xFFFFFFFFu, lA, 2);
    lB += __shfl_xor_sync(0xFFFFFFFFu, lB, 1);
    lB += __shfl_xor_sync(0xFFFFFFFFu, lB, 2);

    // The key warps' parts of the rows are joined in shared memory, warps of
    // the upper half into the lower one, in the last tile's place (tiles behind it
    // may be on their way).
    if constexpr (KW > 1) {
      constexpr int kLane = kOut * 4 + 4;  // values a lane hands over
      float* x = reinterpret_cast<float*>(smem + (kBatch ? (at - 1) % kStages * L::kStage : 0));
      static_assert((size_t)MW * (KW / 2) * 32 * kLane * 4 <= L::kStage, "join fits a tile");
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
    }
    if (kw == 0) {
      // One split: the rows are complete (a row without keys is zeros). Else the
      // parts go to the workspace as they are, in 32 bits.
      const bool whole = !kBatch && a.whole && a.splits == 1;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int r = half ? rB : rA, tok = half ? tB : tA;
        if (r >= R) continue;
        const float m = half ? mB : mA, l = half ? lB : lA;
        const float f = whole ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
        const size_t at = walk.part(a, rows_of, head, parts, r);
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
  } while (kBatch && at < walk.count());
  if constexpr (kBatch) sg::pdl_wait();
}

// Up to kFewRows rows a kv head, fp32, head_dim 128: FMAs. Most of a matrix
// instruction's 16 rows would be empty, and three products of each bound
// k_tree: 4 rows over 8 x 128000 keys take 238 us there, 190 here (5.5 TB/s),
// over 8 x 500 9.4 and 7.9. (With shorter heads a key's softmax outweighs its
// products: 64 entries 111 there, 128 here.) A warp takes 8 keys at a time;
// four lanes share a key's scores, each having a quarter of the entries of key
// and queries, then every lane has 4 entries of the outputs.
constexpr int kFewRows = 4, kFewWarps = 4, kFewHeadDim = 128;

template <typename Args>
__global__ void __launch_bounds__(32 * kFewWarps, 2) k_tree_few(Args a) {
  constexpr int HD = kFewHeadDim;
  constexpr bool kBatch = std::is_same<Args, sg::BatchArgs>::value;
  using L = Tile<float, HD, kFewWarps>;
  constexpr int kWarpKeys = L::kKeys / kFewWarps, kQ = HD / 16, kO = HD / 32;
  static_assert(kWarpKeys == 8, "a warp's keys of a tile are one step");
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
  if constexpr (!kBatch) sg::pdl_wait();  // (see k_tree)
  sg::pdl_trigger();
  using W = Walker<float, HD, 32 * kFewWarps, kFewRows, Args>;
  auto start = [&] {
    if constexpr (kBatch) {
      __shared__ typename W::Shared shared;
      return W(a, shared, smem);
    } else {
      return W(a, smem);
    }
  };
  W walk = start();
  if (walk.count() == 0) {
    if constexpr (kBatch) sg::pdl_wait();
    return;
  }
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) walk.fetch(s);

  int at = 0;  // tiles gone through
  do {
    const Rows rows_of = walk.rows(at);
    const int head = walk.head(at), R = rows_of.t * a.group, parts = walk.parts(at);
    // Scores in units of log2, so that the softmax is exp2.
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    ulonglong2 q[kFewRows][kQ];
    float m[kFewRows], l[kFewRows];
    f32x2 o[kFewRows][kO / 2];
#pragma unroll
    for (int r = 0; r < kFewRows; r++) {
      const int row = r < R ? r : 0, tok = row / a.group;
      const float* from = static_cast<const float*>(a.q) + (rows_of.token0 + tok) * a.ldq +
                          (size_t)(head * a.group + row - tok * a.group) * HD + 4 * c4;
#pragma unroll
      for (int j = 0; j < kQ; j++) {
        const float4 x = *reinterpret_cast<const float4*>(from + 16 * j);
        q[r][j].x = pack2(x.x * scale, x.y * scale);
        q[r][j].y = pack2(x.z * scale, x.w * scale);
      }
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kO / 2; i++) o[r][i] = 0;
    }

    for (bool more = true; more; at++) {
      cp_async_wait<kStages - 2>();
      __syncthreads();
      walk.fetch(at + kStages - 1);  // into the buffer that the last tile left
      int rows, first;
      walk.keys(at, rows, first);
      more = !walk.last(at);
      const bool old = first < 0;
      const unsigned char* ks = smem + at % kStages * L::kStage;
      const unsigned char* vs = ks + L::kKeys * L::kKRow;
      const int k0 = warp * kWarpKeys;  // the warp's first key in the tile
      if (k0 < rows) {
        f32x2 s[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; r++) s[r] = 0;
        const unsigned char* kp = ks + (k0 + g8) * L::kKRow + c4 * 16;
#pragma unroll
        for (int j = 0; j < kQ; j++) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(kp + j * 64);
#pragma unroll
          for (int r = 0; r < kFewRows; r++) {
            s[r] = fma2(q[r][j].x, x.x, s[r]);
            s[r] = fma2(q[r][j].y, x.y, s[r]);
          }
        }
        float p[kFewRows], top[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
          const float2 both = unpack2(s[r]);
          p[r] = both.x + both.y;
          p[r] += __shfl_xor_sync(0xFFFFFFFFu, p[r], 1);
          p[r] += __shfl_xor_sync(0xFFFFFFFFu, p[r], 2);
          bool in = k0 + g8 < rows && r < R;
          if (!old && in) {
            in = seen_of(a, rows_of, r / a.group, first + k0) >> g8 & 1;
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
            for (int i = 0; i < kO / 2; i++) o[r][i] = mul2(pack2(f, f), o[r][i]);
          }
          // A row that has seen no key yet keeps m = -inf and zeros.
          p[r] = exp2f(p[r] - (m[r] == -INFINITY ? 0.f : m[r]));
          l[r] += p[r];
        }
        const unsigned char* vp = vs + k0 * L::kVRow + lane * kO * 4;
#pragma unroll
        for (int kk = 0; kk < 8; kk++) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(vp + kk * L::kVRow);
#pragma unroll
          for (int r = 0; r < kFewRows; r++) {
            const float w = __shfl_sync(0xFFFFFFFFu, p[r], 4 * kk);
            // A drafted row that is hidden may hold anything; cached ones are
            // seen by all.
            if (old || w != 0.f) {
              o[r][0] = fma2(pack2(w, w), x.x, o[r][0]);
              o[r][1] = fma2(pack2(w, w), x.y, o[r][1]);
            }
          }
        }
      }
    }
    if constexpr (!kBatch) cp_async_wait<0>();
    __syncthreads();

    // The warps' parts are joined in shared memory, a row by each warp, in the last
    // tile's place.
    float* part =  // [warp][row][HD + 2]
        reinterpret_cast<float*>(smem + (kBatch ? (at - 1) % kStages * L::kStage : 0));
    static_assert(kFewWarps * kFewRows * (HD + 2) * 4 <= (int)L::kStage, "join fits a tile");
    static_assert(kFewWarps == kFewRows, "a warp per row");
#pragma unroll
    for (int r = 0; r < kFewRows; r++) {
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 4);
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 8);
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 16);
      float* to = part + (warp * kFewRows + r) * (HD + 2);
#pragma unroll
      for (int i = 0; i < kO / 2; i++)
        *reinterpret_cast<float2*>(to + lane * kO + 2 * i) = unpack2(o[r][i]);
      if (lane == 0) {
        to[HD] = m[r];
        to[HD + 1] = l[r];
      }
    }
    __syncthreads();
    if (warp < R) {
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
      const bool whole = !kBatch && a.whole && a.splits == 1;
      const float f = whole ? (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)) : 1.f;
      const int tok = warp / a.group;
      const size_t at = walk.part(a, rows_of, head, parts, warp);
      if (!whole && lane == 0) a.ml[at] = make_float2(all, sum);
      float* to = whole ? static_cast<float*>(a.att) + tok * a.ldo +
                              (size_t)(head * a.group + warp - tok * a.group) * HD
                        : a.part + at * HD;
#pragma unroll
      for (int i = 0; i < kO; i++) to[lane * kO + i] = out[i] * f;
    }
  } while (kBatch && at < walk.count());
  if constexpr (kBatch) sg::pdl_wait();
}

// 2^x; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The transpose of an 8 x 8 matrix of 16-bit values, a row to four lanes.
__device__ __forceinline__ uint32_t transpose(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}

// A batch's own tiles, up to 8 NT rows a request and kv head: the keys are the 16 rows
// of matrix instructions, the queries their columns, so that one token of eight heads
// fills what k_tree's 16 rows would leave half empty, and the scores come out as the
// weights go in. Rows rescale only when a score is 2^8 above what their weights are
// relative to. A warp has the same keys of each tile, 16 or 32 at a time, and all of the
// outputs or (fp32, 128 entries, where a tile has 32 keys) half of them.
//   S^T = K Q^T;  O^T += V^T P^T
// fp32: tf32 parts as in k_tree. A matrix instruction cuts its sums, so those of small
// products and of large ones are kept apart, and outputs start from zero at each step
// and are added with rounding. Entries of a row, and keys, are numbered so that a lane's
// are neighbours: any order serves, if both operands have it.
constexpr int kOwnWarps = 4;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(32 * kOwnWarps, 2) k_own(sg::BatchArgs a) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kThreads = 32 * kOwnWarps, kRows = 8 * NT;
  using L = Tile<T, HD, kOwnWarps>;
  // Warps side by side in keys, and in outputs.
  constexpr int kKeys = L::kKeys, kSide = kKeys / 16 < kOwnWarps ? kKeys / 16 : kOwnWarps;
  constexpr int kShares = kOwnWarps / kSide, kWarpKeys = kKeys / kSide;
  constexpr int kStep = NT > 2 || kWarpKeys < 32 ? 16 : 32, kGroups = kStep / 16;
  constexpr int kQ = HD / 16, kO = kQ / kShares;  // 16 entries: of the scores, of a warp's outputs
  static_assert(!kF32 || kGroups == 1, "16 keys a step");
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
  sg::pdl_trigger();  // (see k_tree)
  const int side = warp % kSide, share = warp / kSide;
  using W = Stream<T, HD, kThreads, kRows>;
  __shared__ typename W::Shared shared;
  W walk(a, shared, smem);
  if (walk.count() == 0) {
    sg::pdl_wait();
    return;
  }
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) walk.fetch(s);
  const float scale = 1.4426950408889634f / sqrtf((float)HD);  // scores in units of log2

  // r / group: mul is above 2^16 / group by 1 at most, which r < 64 does not carry into
  // the quotient.
  static_assert(kRows <= 64, "all rows of a request");
  const unsigned mul = 65536u / a.group + 1;
  auto token = [&](int r) { return (int)(r * mul >> 16); };

  int at = 0;  // tiles gone through
  do {
    const Rows rows_of = walk.rows(at);
    const int head = walk.head(at), R = rows_of.t * a.group, r0 = rows_of.r0;
    const int parts = walk.parts(at);
    auto query = [&](int r) {  // of row r of the request
      const int tok = token(r);
      return static_cast<const T*>(a.q) + (rows_of.token0 + tok) * a.ldq +
             (size_t)(head * a.group + r - tok * a.group) * HD;
    };
    // bf16: operands as they are; fp32: the parts of entries 16 k + 4 c4 + {0, 1} and
    // {2, 3}.
    uint32_t q[NT][kQ][kF32 ? 8 : 2];
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int r = r0 + 8 * j + g8;
      const T* const from = query(r < R ? r : r0) + (kF32 ? 4 : 2) * c4;
#pragma unroll
      for (int k = 0; k < kQ; k++) {
        if constexpr (kF32) {
          const float4 x = r < R ? *reinterpret_cast<const float4*>(from + 16 * k)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
          split_tf32(x.x, q[j][k][0], q[j][k][4]);
          split_tf32(x.y, q[j][k][1], q[j][k][5]);
          split_tf32(x.z, q[j][k][2], q[j][k][6]);
          split_tf32(x.w, q[j][k][3], q[j][k][7]);
        } else {
#pragma unroll
          for (int h = 0; h < 2; h++)
            q[j][k][h] = r < R ? *reinterpret_cast<const uint32_t*>(from + 16 * k + 8 * h) : 0u;
        }
      }
    }
    // This lane's rows 8 j + 2 c4 + e: their last drafted key, maximum and (this
    // lane's keys') sum; outputs entry(i, h) of them.
    auto entry = [&](int i, int h) {
      return kF32 ? share * (HD / kShares) + 32 * (i / 2) + 4 * g8 + i % 2 * 2 + h
                  : 16 * i + g8 + 8 * h;
    };
    int last[NT][2];
    float m[NT][2], l[NT][2], o[NT][kO][4];
#pragma unroll
    for (int j = 0; j < NT; j++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = r0 + 8 * j + 2 * c4 + e;
        last[j][e] = r < R ? token(r) - rows_of.late : -1;
        m[j][e] = -INFINITY;
        l[j][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kO; i++) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    }

    for (bool more = true; more; at++) {
      cp_async_wait<kStages - 2>();
      __syncthreads();
      walk.fetch(at + kStages - 1);  // into the buffer that the last tile left
      int rows, first;
      walk.keys(at, rows, first);
      more = !walk.last(at);
      const unsigned char* ks = smem + at % kStages * L::kStage;
      const unsigned char* vs = ks + kKeys * L::kKRow;
      // As in k_tree: an infinity or NaN in a value row that some rows do not see.
      bool slow = false;
      if (first >= 0) {
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
      for (int ch = 0; ch < kWarpKeys; ch += kStep) {
        const int k0 = side * kWarpKeys + ch;  // first key of the step in the tile
        if (k0 >= rows) break;
        float s[NT][kGroups][4];
        if constexpr (kF32) {
          float big[NT][2][4], small[NT][2][4];
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int x = 0; x < 8; x++) (&big[j][0][0])[x] = (&small[j][0][0])[x] = 0.f;
          const unsigned char* const kp = ks + (k0 + g8) * L::kKRow + c4 * 16;
#pragma unroll
          for (int k = 0; k < kQ; k++) {
            const float4 x = *reinterpret_cast<const float4*>(kp + k * 64);
            const float4 y = *reinterpret_cast<const float4*>(kp + 8 * L::kKRow + k * 64);
            uint32_t hi[2][4], lo[2][4];
            split_tf32(x.x, hi[0][0], lo[0][0]);
            split_tf32(y.x, hi[0][1], lo[0][1]);
            split_tf32(x.y, hi[0][2], lo[0][2]);
            split_tf32(y.y, hi[0][3], lo[0][3]);
            split_tf32(x.z, hi[1][0], lo[1][0]);
            split_tf32(y.z, hi[1][1], lo[1][1]);
            split_tf32(x.w, hi[1][2], lo[1][2]);
            split_tf32(y.w, hi[1][3], lo[1][3]);
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const uint32_t* const w = q[j][k] + 2 * h;
                mma_tf32(small[j][h], lo[h], w[0], w[1]);
                mma_tf32(big[j][h], hi[h], w[0], w[1]);
                mma_tf32(small[j][h], hi[h], w[4], w[5]);
              }
          }
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int x = 0; x < 4; x++)
              s[j][0][x] = (small[j][0][x] + small[j][1][x]) + (big[j][0][x] + big[j][1][x]);
        } else {
          const uint32_t kp = saddr(ks) + (k0 + (lane & 15)) * L::kKRow + (lane >> 4) * 16;
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int b = 0; b < kGroups; b++)
              s[j][b][0] = s[j][b][1] = s[j][b][2] = s[j][b][3] = 0.f;
#pragma unroll
          for (int k = 0; k < kQ; k++)
#pragma unroll
            for (int b = 0; b < kGroups; b++) {
              uint32_t x[4];
              ldsm4(kp + b * 16 * L::kKRow + k * 32, x);
#pragma unroll
              for (int j = 0; j < NT; j++) mma_bf16(s[j][b], x, q[j][k][0], q[j][k][1]);
            }
        }
        // What the rows do not see.
        if (first >= 0 || k0 + kStep > rows) {
#pragma unroll
          for (int b = 0; b < kGroups; b++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
              const int key = k0 + 16 * b + g8 + 8 * (x >> 1);
#pragma unroll
              for (int j = 0; j < NT; j++)
                if (key >= rows || (first >= 0 && first + key > last[j][x & 1]))
                  s[j][b][x] = -INFINITY;
            }
        }
        // A new maximum, for all lanes of a row.
        float top[NT][2];
        bool higher = false;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float x = fmaxf(s[j][0][e], s[j][0][2 + e]);
#pragma unroll
            for (int b = 1; b < kGroups; b++) x = fmaxf(x, fmaxf(s[j][b][e], s[j][b][2 + e]));
            top[j][e] = x * scale;
            higher = higher || top[j][e] > m[j][e] + 8.f;
          }
        if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float x = top[j][e];
#pragma unroll
              for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
              const float next = fmaxf(m[j][e], x);
              // A row that has seen no key yet keeps m = -inf and zeros.
              const float f = next == -INFINITY ? 1.f : ex2(m[j][e] - next);
              m[j][e] = next;
              l[j][e] *= f;
#pragma unroll
              for (int i = 0; i < kO; i++) {
                o[j][i][e] *= f;
                o[j][i][2 + e] *= f;
              }
            }
        }
        // Weights, as two bf16 parts, or tf32 parts; transposed, they are operands.
        uint32_t ph[NT][kGroups][kF32 ? 4 : 2], pl[NT][kGroups][kF32 ? 4 : 2];
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const float z0 = m[j][0] == -INFINITY ? 0.f : m[j][0];
          const float z1 = m[j][1] == -INFINITY ? 0.f : m[j][1];
#pragma unroll
          for (int b = 0; b < kGroups; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float& x = s[j][b][2 * h];
              float& y = s[j][b][2 * h + 1];
              x = ex2(fmaf(x, scale, -z0));
              y = ex2(fmaf(y, scale, -z1));
              l[j][0] += x;
              l[j][1] += y;
              if constexpr (kF32) {
                // Upper and lower halves; then keys 8 h + 2 c4 and the next one.
                const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
                const uint32_t up = transpose(__byte_perm(u, v, 0x7632));
                const uint32_t down = transpose(__byte_perm(u, v, 0x5410));
                split_tf32(__uint_as_float(__byte_perm(down, up, 0x5410)), ph[j][b][2 * h],
                           pl[j][b][2 * h]);
                split_tf32(__uint_as_float(__byte_perm(down, up, 0x7632)), ph[j][b][2 * h + 1],
                           pl[j][b][2 * h + 1]);
              } else {
                uint32_t hi, lo;
                split_bf16(x, y, hi, lo);
                ph[j][b][h] = transpose(hi);
                pl[j][b][h] = transpose(lo);
              }
            }
        }
        if (slow) {
          // Key by key, weights of exactly 0 left out.
          for (int kk = 0; kk < kStep && k0 + kk < rows; kk++) {
            const T* const row = reinterpret_cast<const T*>(vs + (k0 + kk) * L::kVRow);
#pragma unroll
            for (int j = 0; j < NT; j++) {
              float w[2] = {0.f, 0.f};
#pragma unroll
              for (int b = 0; b < kGroups; b++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                  if (kk / 8 == 2 * b + h) {
                    w[0] = s[j][b][2 * h];
                    w[1] = s[j][b][2 * h + 1];
                  }
              const int from = kk % 8 * 4 + c4;
              w[0] = __shfl_sync(0xFFFFFFFFu, w[0], from);
              w[1] = __shfl_sync(0xFFFFFFFFu, w[1], from);
#pragma unroll
              for (int i = 0; i < kO; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                  if (w[x & 1] == 0.f) continue;
                  const T v = row[entry(i, x >> 1)];
                  if constexpr (kF32)
                    o[j][i][x] = fmaf(w[x & 1], v, o[j][i][x]);
                  else
                    o[j][i][x] = fmaf(w[x & 1], sg::bf16_to_f32(v), o[j][i][x]);
                }
            }
          }
          continue;
        }
        if constexpr (kF32) {
          const unsigned char* const vp =
              vs + (k0 + 2 * c4) * L::kVRow + (share * (HD / kShares) + 4 * g8) * 4;
#pragma unroll
          for (int i = 0; i < kO; i += 2) {
            uint32_t hi[2][2][4], lo[2][2][4];  // [half of the keys][tile]
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const unsigned char* const p = vp + 8 * h * L::kVRow + i * 64;
              const float4 x = *reinterpret_cast<const float4*>(p);
              const float4 y = *reinterpret_cast<const float4*>(p + L::kVRow);
              split_tf32(x.x, hi[h][0][0], lo[h][0][0]);
              split_tf32(x.y, hi[h][0][1], lo[h][0][1]);
              split_tf32(y.x, hi[h][0][2], lo[h][0][2]);
              split_tf32(y.y, hi[h][0][3], lo[h][0][3]);
              split_tf32(x.z, hi[h][1][0], lo[h][1][0]);
              split_tf32(x.w, hi[h][1][1], lo[h][1][1]);
              split_tf32(y.z, hi[h][1][2], lo[h][1][2]);
              split_tf32(y.w, hi[h][1][3], lo[h][1][3]);
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
              for (int t = 0; t < 2; t++) {
                const uint32_t *const wh = ph[j][0], *const wl = pl[j][0];
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                mma_tf32(y, lo[0][t], wh[0], wh[1]);
                mma_tf32(y, lo[1][t], wh[2], wh[3]);
                mma_tf32(y, hi[0][t], wl[0], wl[1]);
                mma_tf32(y, hi[1][t], wl[2], wl[3]);
                mma_tf32(y, hi[0][t], wh[0], wh[1]);
                mma_tf32(y, hi[1][t], wh[2], wh[3]);
#pragma unroll
                for (int x = 0; x < 4; x++) o[j][i + t][x] += y[x];
              }
          }
        } else {
          const uint32_t vp = saddr(vs) + (k0 + (lane & 7) + (lane >> 4) * 8) * L::kVRow +
                              ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int b = 0; b < kGroups; b++)
#pragma unroll
            for (int i = 0; i < kO; i++) {
              uint32_t x[4];
              ldsm4t(vp + b * 16 * L::kVRow + i * 32, x);
#pragma unroll
              for (int j = 0; j < NT; j++) {
                mma_bf16(o[j][i], x, pl[j][b][0], pl[j][b][1]);
                mma_bf16(o[j][i], x, ph[j][b][0], ph[j][b][1]);
              }
            }
        }
      }
    }

    // The warps' parts are joined in shared memory, in the last tile's place (tiles
    // behind it may be on their way), kAtOnce tiles of rows at a time: every warp
    // hands over all that it has, and adds up a quarter of the outputs.
    constexpr int kLane = 4 * kO + 4;  // values a lane hands over per tile of rows
    constexpr int kFits = L::kStage / (kOwnWarps * 32 * kLane * 4);
    constexpr int kAtOnce = kFits < NT ? kFits : NT, kApart = 32 * kOwnWarps;
    static_assert(kAtOnce > 0, "a tile of rows fits");
    // [value][warp][lane]: lanes side by side.
    float* const x = reinterpret_cast<float*>(smem + (at - 1) % kStages * L::kStage);
#pragma unroll
    for (int j0 = 0; j0 < NT; j0 += kAtOnce) {
      __syncthreads();
#pragma unroll
      for (int j = j0; j < j0 + kAtOnce && j < NT; j++) {
        float* p = x + (j - j0) * kLane * kApart + threadIdx.x;
#pragma unroll
        for (int i = 0; i < kO; i++)
#pragma unroll
          for (int e = 0; e < 4; e++, p += kApart) *p = o[j][i][e];
#pragma unroll
        for (int e = 0; e < 2; e++, p += 2 * kApart) {
#pragma unroll
          for (int d = 4; d < 32; d *= 2) l[j][e] += __shfl_xor_sync(0xFFFFFFFFu, l[j][e], d);
          p[0] = m[j][e];
          p[kApart] = l[j][e];
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = j0; j < j0 + kAtOnce && j < NT; j++) {
        const float* const p = x + (j - j0) * kLane * kApart + lane;
        float f[2][kSide];
        float* to[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float* const ml = p + (4 * kO + 2 * e) * kApart;
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kSide; w++) top = fmaxf(top, ml[32 * w]);
#pragma unroll
          for (int w = 0; w < kSide; w++) {
            f[e][w] = top == -INFINITY ? 0.f : ex2(ml[32 * w] - top);
            sum += f[e][w] * ml[kApart + 32 * w];
          }
          const int r = r0 + 8 * j + 2 * c4 + e;
          const size_t at_row = r < R ? walk.part(a, rows_of, head, parts, r) : 0;
          to[e] = r < R ? a.part + at_row * HD : nullptr;
          if (r < R && g8 == 0 && warp == 0) a.ml[at_row] = make_float2(top, sum);
        }
        auto sum_of = [&](int e, int value, int from) {  // of warps `from` on
          const float* const v = p + value * kApart + 32 * from;
          float y = 0.f;
#pragma unroll
          for (int w = 0; w < kSide; w++) y = fmaf(f[e][w], v[32 * w], y);
          return y;
        };
        if constexpr (kF32) {
          // 32 entries, four to a lane.
          if (warp < HD / 32) {
            const int from = warp / (kO / 2) * kSide, i = warp % (kO / 2) * 8;
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float4 y =
                  make_float4(sum_of(e, i + e, from), sum_of(e, i + 2 + e, from),
                              sum_of(e, i + 4 + e, from), sum_of(e, i + 6 + e, from));
              if (to[e]) *reinterpret_cast<float4*>(to[e] + 32 * warp + 4 * g8) = y;
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2 * kO; u += kOwnWarps) {
            const int of = u + warp;  // outputs 8 of + g8
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float y = sum_of(e, of / 2 * 4 + of % 2 * 2 + e, 0);
              if (to[e]) to[e][8 * of + g8] = y;
            }
          }
        }
      }
    }
  } while (at < walk.count());
  sg::pdl_wait();
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
                    (DRAFTED ? 0 : (a.drafted + keys_per_tile - 1) / keys_per_tile);
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

// A batch's parts: those of the prefix, that of the run with the row's first own
// tile, those of the runs that go on with it. WARPS of a block share a row, a run of
// its parts each: a lane has a part's maximum and sum, then HD / 32 entries of the
// outputs. Rows of no request stay as they are.
struct JoinArgs : TreeArgs {   // of the prefix
  const int2* where;
  int ctas, rows;              // of the requests' own tiles: CTAs, and rows of one
  int requests, most;
  const int* first;
};
constexpr int kJoinWarps = 4;
constexpr int kJoinFew = 4096;  // rows for which a block each is on its way at once

template <typename T, int HD, int WARPS>
__global__ void __launch_bounds__(32 * kJoinWarps) k_join(JoinArgs a, int keys_per_tile) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part_of = warp % WARPS;
  // (Rows are fewer than 2^31; parts that a GPU's memory holds, than 2^32.)
  const unsigned all = (unsigned)a.t * a.group, rows = all * a.kh;
  const unsigned row = blockIdx.x * (kJoinWarps / WARPS) + warp / WARPS;
  const unsigned head = row / all, r = row - head * all;
  const int tok = (int)(r / (unsigned)a.group);
  sg::pdl_trigger();
  sg::pdl_wait();
  const bool in = row < rows && (a.first ? tok >= a.first[0] && tok < a.first[a.requests]
                                         : tok < (long long)a.requests * a.most);
  if (WARPS == 1 && !in) return;
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; i++) o[i] = 0.f;
  if (in) {
    const unsigned tiles = (sg::tree_cached(a) + keys_per_tile - 1) / keys_per_tile;
    const unsigned per = (tiles + a.splits - 1) / a.splits;
    const int prefix = tiles ? (int)((tiles + per - 1) / per) : 0;
    // (Within the workspace, whatever stands there.)
    const int2 w = a.where[row];
    const int cta = min(max(w.x, 0), a.ctas - 1), place = min(w.y & 127, a.rows - 1);
    const int parts = prefix + min(max(w.y >> 7, 1), a.ctas - cta);
    const int share = (parts + WARPS - 1) / WARPS, end = min(parts, (part_of + 1) * share);
    for (int from = part_of * share; from < end; from += 32) {
      const int n = min(32, end - from), i = from + lane;  // i: this lane's part
      const unsigned at = i <= prefix ? (i < prefix ? i : a.splits) * rows + row
                                      : (a.splits + 1) * rows + (cta + i - prefix) * a.rows + place;
      const float2 p = lane < n ? a.ml[at] : make_float2(-INFINITY, 0.f);
      const float next = fmaxf(m, sg::warp_max(p.x));
      const float f = next == -INFINITY ? 1.f : exp2f(m - next);
      const float g = next == -INFINITY || p.y == 0.f ? 0.f : exp2f(p.x - next);
      m = next;
      l = l * f + sg::warp_sum(p.y == 0.f ? 0.f : p.y * g);
#pragma unroll
      for (int v = 0; v < V; v++) o[v] *= f;
#pragma unroll 4
      for (int j = 0; j < n; j++) {
        const float weight = __shfl_sync(0xFFFFFFFFu, g, j);
        const float* x = a.part + (size_t)__shfl_sync(0xFFFFFFFFu, at, j) * HD + lane * V;
        float y[V];
        if constexpr (V == 4) {
          const float4 z = *reinterpret_cast<const float4*>(x);
          y[0] = z.x; y[1] = z.y; y[2] = z.z; y[3] = z.w;
        } else if constexpr (V == 2) {
          const float2 z = *reinterpret_cast<const float2*>(x);
          y[0] = z.x; y[1] = z.y;
        } else {
          y[0] = *x;
        }
        // Weight 0: no keys, or too far below; the part may hold anything.
#pragma unroll
        for (int v = 0; v < V; v++) o[v] = weight == 0.f ? o[v] : fmaf(weight, y[v], o[v]);
      }
    }
  }
  if constexpr (WARPS > 1) {
    __shared__ float outs[kJoinWarps][HD];
    __shared__ float2 sums[kJoinWarps];
#pragma unroll
    for (int i = 0; i < V; i++) outs[warp][lane * V + i] = o[i];
    if (lane == 0) sums[warp] = make_float2(m, l);
    __syncthreads();
    if (part_of || !in) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, sums[warp + w].x);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = top == -INFINITY ? 0.f : exp2f(sums[warp + w].x - top);
      l += sums[warp + w].y * f;
#pragma unroll
      for (int i = 0; i < V; i++) o[i] = fmaf(outs[warp + w][lane * V + i], f, o[i]);
    }
  }
  // A row without keys is zeros.
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* to = static_cast<T*>(a.att) + tok * a.ldo + (size_t)(head * a.group + r - tok * a.group) * HD +
          lane * V;
  union {
    T entry[V];
    std::conditional_t<V * sizeof(T) == 16, uint4,
        std::conditional_t<V * sizeof(T) == 8, uint2,
            std::conditional_t<V * sizeof(T) == 4, uint32_t, uint16_t>>> all;
  } out;
#pragma unroll
  for (int i = 0; i < V; i++) {
    if constexpr (sizeof(T) == 4)
      out.entry[i] = o[i] * f;
    else
      asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(out.entry[i]) : "f"(o[i] * f));
  }
  *reinterpret_cast<decltype(out.all)*>(to) = out.all;
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

// Whether fp32 rows go to k_tree_few.
bool few_rows(int hd, int rows) { return hd == kFewHeadDim && rows <= kFewRows; }

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

// Tiles of eight rows of k_own that take a request's `rows`; 0: k_tree (or k_tree_few)
// takes them. Measured with 8 kv heads behind a prefix of 64 rows, us of a call with k_own /
// k_tree, for 48 requests of 1000 rows, 8 of 4000 and 16 of 200:
//   head_dim 128,  4 rows: 49 / 57, 36 / 42, 13.3 / 15.8
//                 16 rows: 60 / 61, 44 / 45, 18.7 / 18.4
//   head_dim 64,   8 rows: 34 / 41, 21 / 26, 13.5 / 15.9
//                 16 rows: 37 / 40, 26 / 28, 16.0 / 16.7
//                 32 rows: 52 / 54, 34 / 34, 22.9 / 20.5
//                 48 rows: 76 / 73, 46 / 51, 25.3 / 18.9
//   head_dim 32,  32 rows: 42 / 48, 29 / 33, 20.5 / 18.2
//                 48 rows: 57 / 73, 38 / 48, 20.7 / 16.6
// (k_tree takes 48 rows as 64.) Where neither is always ahead, it goes by the longer
// ones. fp32, k_own / k_tree or (128 entries, 4 rows) k_tree_few:
//   head_dim 128,  4 rows: 111 / 105, 87 / 79, 16.9 / 17.9
//                  8 rows: 115 / 141, 86 / 105, 20.0 / 22.4
//                 16 rows: 146 / 145, 111 / 109, 23.1 / 25.4
//   head_dim 64,   8 rows: 61 / 73, 45 / 54, 15.3 / 17.3
//                 16 rows: 72 / 73, 56 / 56, 17.5 / 17.8
//   head_dim 32,   8 rows: 44 / 53, 29 / 36, 13.0 / 13.7
//                 16 rows: 52 / 52, 37 / 37, 15.7 / 15.6
int own_tiles(int hd, bool f32, int rows) {
  if (f32) return rows > 8 || few_rows(hd, rows) ? 0 : 1;
  if (rows <= 8) return 1;
  if (rows <= 16) return 2;
  if (rows <= 32) return hd == 32 ? 4 : 0;
  return rows <= 48 && hd < 128 ? 6 : 0;
}
// Rows of a tile of requests' rows.
int own_rows(int hd, bool f32, int rows) {
  if (f32 && few_rows(hd, rows)) return kFewRows;
  const int tiles = own_tiles(hd, f32, rows);
  return tiles ? 8 * tiles : 16 * shape_of(rows).mw;
}

// Whether a shared prefix's keys go to tcgen05: on_tc's rule, whatever the tokens.
bool prefix_on_tc(int rows, int hd) { return hd >= 64 && rows > (hd == 128 ? 16 : 32); }

// Splits of the keys: as many CTAs as the GPU holds at once.
int splits_of(int sms, int rows, int kh, bool tc) {
  const Shape s = shape_of(rows);
  const int resident = sms * (!tc && s.mw * s.kw <= 4 ? 2 : 1);
  const int tile = tc ? sg::kTreeTcRows : 16 * s.mw;
  const long long others = (long long)kh * ((rows + tile - 1) / tile);
  return (int)std::max(1ll, std::min((long long)kMaxSplits, resident / others));
}

size_t workspace_of(int splits, int t, int kh, int group, int hd) {
  if (splits == 1 && !on_tc(t, group, hd)) return 0;
  return (size_t)splits * kh * t * group * (hd + 2) * sizeof(float);
}

// CTAs for the splits and row tiles of a tree; of a batch.
dim3 grid_of(const TreeArgs& a, int tile_rows) {
  return dim3(a.splits, a.kh, (a.t * a.group + tile_rows - 1) / tile_rows);
}
dim3 grid_of(const sg::BatchArgs& a, int) { return dim3(a.ctas); }

template <typename Args>
cudaError_t launch_few(const Args& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  using L = Tile<float, kFewHeadDim, kFewWarps>;
  const cudaError_t e = sg::allow_smem(k_tree_few<Args>, L::kBytes, dev, allowed);
  if (e != cudaSuccess) return e;
  return sg::try_launch(k_tree_few<Args>, grid_of(a, kFewRows), dim3(32 * kFewWarps), L::kBytes, 1,
                        s, a);
}

template <typename T, int HD, int MW, int KW, typename Args>
cudaError_t launch_shape(const Args& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  constexpr size_t bytes = Tile<T, HD, MW * KW>::kBytes;
  const cudaError_t e = sg::allow_smem(k_tree<T, HD, MW, KW, Args>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  return sg::try_launch(k_tree<T, HD, MW, KW, Args>, grid_of(a, 16 * MW), dim3(32 * MW * KW), bytes,
                        1, s, a);
}

// This file's kernels for `rows` rows of a kv head (of a tree, of a request);
// *keys: of a tile of theirs.
template <typename T, int HD>
cudaError_t launch_mma(const TreeArgs& a, int rows, int* keys, int dev, cudaStream_t s) {
  if constexpr (sizeof(T) == 4 && HD == kFewHeadDim)
    if (few_rows(HD, rows)) {
      *keys = Tile<float, HD, kFewWarps>::kKeys;
      return launch_few(a, dev, s);
    }
  const Shape f = shape_of(rows);
  *keys = f.mw * f.kw <= 4 ? Tile<T, HD, 4>::kKeys : Tile<T, HD, 8>::kKeys;
  if (f.mw == 1) return launch_shape<T, HD, 1, 4>(a, dev, s);
  if (f.mw == 2) return launch_shape<T, HD, 2, 2>(a, dev, s);
  if (f.mw == 4) return launch_shape<T, HD, 4, 1>(a, dev, s);
  return launch_shape<T, HD, 8, 1>(a, dev, s);
}

template <typename T, int HD>
cudaError_t launch_hd(const TreeArgs& a, int dev, cudaStream_t s) {
  const dim3 rows(a.t * a.group * a.kh);
  if (on_tc(a.t, a.group, HD)) {
    if constexpr (HD >= 64) {
      constexpr bool kF32 = sizeof(T) == 4;
      const cudaError_t e = sg::tree_tc(a, kF32, HD, dev, s);
      if (e != cudaSuccess) return e;
      return sg::try_launch(k_merge<T, HD, true>, rows, dim3(kMergeThreads), 0, 1, s, a,
                            sg::tree_tc_keys());
    }
  }
  int keys = 0;
  const cudaError_t e = launch_mma<T, HD>(a, a.t * a.group, &keys, dev, s);
  if (e != cudaSuccess || a.splits == 1) return e;
  return sg::try_launch(k_merge<T, HD, false>, rows, dim3(kMergeThreads), 0, 1, s, a, keys);
}

template <typename T, int HD, int NT>
cudaError_t launch_own_as(const sg::BatchArgs& a, int dev, cudaStream_t s) {
  static std::atomic<size_t> allowed[sg::kDevices];
  constexpr size_t bytes = Tile<T, HD, kOwnWarps>::kBytes;
  const cudaError_t e = sg::allow_smem(k_own<T, HD, NT>, bytes, dev, allowed);
  if (e != cudaSuccess) return e;
  return sg::try_launch(k_own<T, HD, NT>, dim3(a.ctas), dim3(32 * kOwnWarps), bytes, 1, s, a);
}

// A batch's own tiles.
template <typename T, int HD>
cudaError_t launch_own(const sg::BatchArgs& a, int dev, cudaStream_t s) {
  const int rows = a.most * a.group, tiles = own_tiles(HD, sizeof(T) == 4, rows);
  if (tiles == 1) return launch_own_as<T, HD, 1>(a, dev, s);
  if constexpr (sizeof(T) == 2)
    if (tiles == 2) return launch_own_as<T, HD, 2>(a, dev, s);
  if constexpr (sizeof(T) == 2 && HD == 32)
    if (tiles == 4) return launch_own_as<T, HD, 4>(a, dev, s);
  if constexpr (sizeof(T) == 2 && HD < 128)
    if (tiles == 6) return launch_own_as<T, HD, 6>(a, dev, s);
  const int mw = shape_of(rows).mw;
  if constexpr (sizeof(T) == 4) {
    if constexpr (HD == kFewHeadDim)
      if (few_rows(HD, rows)) return launch_few(a, dev, s);
    if (mw == 1) return launch_shape<T, HD, 1, 4>(a, dev, s);
  }
  if constexpr (sizeof(T) == 4 || HD > 32)
    if (mw == 2) return launch_shape<T, HD, 2, 2>(a, dev, s);
  return mw == 4 ? launch_shape<T, HD, 4, 1>(a, dev, s) : launch_shape<T, HD, 8, 1>(a, dev, s);
}

// Behind a shared prefix: parts of the prefix for all rows, parts of each
// request's own keys, and their joins.
template <typename T, int HD>
cudaError_t launch_shared(const TreeArgs& p, const sg::BatchArgs& own, int dev, cudaStream_t s) {
  int keys = 0;
  cudaError_t e;
  if (prefix_on_tc(p.t * p.group, HD)) {
    if constexpr (HD >= 64) e = sg::tree_tc(p, sizeof(T) == 4, HD, dev, s);
    keys = sg::tree_tc_keys();
  } else {
    e = launch_mma<T, HD>(p, p.t * p.group, &keys, dev, s);
  }
  if (e != cudaSuccess) return e;
  e = launch_own<T, HD>(own, dev, s);
  if (e != cudaSuccess) return e;
  JoinArgs j;
  static_cast<TreeArgs&>(j) = p;
  j.where = own.where;
  j.ctas = own.ctas;
  j.rows = own_rows(HD, sizeof(T) == 4, own.most * own.group);
  j.requests = own.requests;
  j.most = own.most;
  j.first = own.first;
  const long long rows = (long long)p.t * p.group * p.kh;
  if (rows <= kJoinFew)
    return sg::try_launch(k_join<T, HD, kJoinWarps>, dim3((unsigned)rows), dim3(32 * kJoinWarps), 0,
                          1, s, j, keys);
  return sg::try_launch(k_join<T, HD, 1>, dim3((unsigned)((rows + kJoinWarps - 1) / kJoinWarps)),
                        dim3(32 * kJoinWarps), 0, 1, s, j, keys);
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

// How a batch is split: its prefix, and the requests' own keys; its workspace.
struct Batch {
  int splits, ctas;
  size_t parts, where, bytes;  // parts; bytes before the notes where they lie, and in all
};
Batch batch_of(int sms, int type, int t, int tokens, int kh, int group, int hd) {
  Batch b;
  const size_t rows = (size_t)kh * tokens * group;
  const bool tc = prefix_on_tc(tokens * group, hd);
  b.splits = splits_of(sms, tokens * group, kh, tc);
  if (tc) {
    // One CTA to an SM: whole rounds of them, in units of a tile's time, for a
    // prefix of 128 tiles (its length is not known here); a CTA's start and end cost
    // as much as six. (16 splits at most: one kv head, 93 fp32 rows of 64 entries over 64543,
    // 115 us, now 37.)
    const int tiles = (tokens * group + sg::kTreeTcRows - 1) / sg::kTreeTcRows;
    const long long units = (long long)kh * tiles;
    double best = 1e30;
    for (int n = 1; n <= kMaxSplits; n++) {
      const double cost = (double)((units * n + sms - 1) / sms) * (128.0 / n + 6);
      if (cost < best) {
        best = cost;
        b.splits = n;
      }
    }
  }
  // As many CTAs as an SM takes (k_own has four warps).
  const Shape s = shape_of(t * group);
  const bool own = own_tiles(hd, type == STRASGPT_F32, t * group) > 0;
  b.ctas = sms * (own || s.mw * s.kw <= kOwnWarps ? 2 : 1);
  b.parts = (b.splits + 1) * rows + (size_t)b.ctas * own_rows(hd, type == STRASGPT_F32, t * group);
  b.where = b.parts * (hd + 2) * sizeof(float);
  b.bytes = b.where + rows * sizeof(int2);
  return b;
}

const char* bad_batch(int type, int requests, int t, int tokens, int kh, int group, int hd) {
  if (type != STRASGPT_F32 && type != STRASGPT_BF16) return "unknown type";
  if (requests < 0 || t <= 0 || tokens < 0 || kh <= 0 || group <= 0) return "empty shape";
  if (t > STRASGPT_ATTN_SHARED_MAX) return "more than 1024 new tokens of a request";
  if (group > 128 || kh > 65535) return "more than 128 q heads per kv head, or 65535 kv heads";
  if (hd != 32 && hd != 64 && hd != 128) return "head_dim must be 32, 64 or 128";
  // k_join has a block per row, the prefix's kernels one per 16 rows or more along
  // z.
  if ((long long)tokens * kh * group > INT_MAX) return "more than 2^31 - 1 rows of q heads";
  if ((long long)tokens * group > 65535ll * 64) return "more than 4194240 rows of a kv head";
  if (requests >= 1 << 30) return "more than 2^30 - 1 requests";
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
  const int splits = splits_of(sms, t * group, kv_heads, on_tc(t, group, head_dim));
  return t ? workspace_of(splits, t, kv_heads, group, head_dim) : 0;
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
  const int splits = splits_of(sms, t * group, kv_heads, on_tc(t, group, head_dim));
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
  a.t = a.drafted = t;
  a.kh = kv_heads; a.group = group; a.ctx = ctx; a.words = (t + 63) / 64;
  a.whole = true;
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

size_t strasgpt_k_attn_shared_workspace(int type, int requests, int t, int tokens, int kv_heads,
                                        int group, int head_dim) {
  const char* const me = "strasgpt_k_attn_shared_workspace";
  if (const char* why = bad_batch(type, requests, t, tokens, kv_heads, group, head_dim)) {
    sg::refuse(me, why);
    return 0;
  }
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) {
    sg::refuse(me, why);
    return 0;
  }
  if (requests == 0 || tokens == 0) return 0;
  return batch_of(sms, type, t, tokens, kv_heads, group, head_dim).bytes;
}

int strasgpt_k_attn_shared(const void* q, long long ldq, const void* k_prefix,
                           const void* v_prefix, int prefix_ctx, const int* prefix,
                           const void* k_cache, const void* v_cache, long long request_stride,
                           int ctx, const int* rows, const int* first, int type, int requests,
                           int t, int tokens, int kv_heads, int group, int head_dim, void* att,
                           long long ldo, void* workspace, size_t workspace_bytes, void* stream) {
  const char* const me = "strasgpt_k_attn_shared";
  if (const char* why = bad_batch(type, requests, t, tokens, kv_heads, group, head_dim))
    return sg::refuse(me, why);
  if (prefix_ctx < 1 || ctx < 1) return sg::refuse(me, "a cache without rows");
  const long long row = (long long)kv_heads * group * head_dim;
  if (tokens > 1 && (ldq < row || ldo < row)) return sg::refuse(me, "rows of q or att overlap");
  if (request_stride < 0) return sg::refuse(me, "negative stride");
  if (requests == 0 || tokens == 0) return 0;
  if (!q || !k_prefix || !v_prefix || !prefix || !k_cache || !v_cache || !rows || !att)
    return sg::refuse(me, "null buffer");
  const size_t size = type == STRASGPT_F32 ? 4 : 2;
  if (!sg::aligned(q, 16) || !sg::aligned(k_prefix, 16) || !sg::aligned(v_prefix, 16) ||
      !sg::aligned(k_cache, 16) || !sg::aligned(v_cache, 16) || !sg::aligned(att, 16) ||
      (tokens > 1 && (ldq * size % 16 || ldo * size % 16)) ||
      (requests > 1 && request_stride * size % 16))
    return sg::refuse(me, "q, the caches, att and their rows must be 16-byte aligned");
  if (q == att && tokens > 1 && ldq != ldo)
    return sg::refuse(me, "in place, q and att must have the same strides");
  if (!sg::aligned(prefix, 4) || !sg::aligned(rows, 4) || !sg::aligned(first, 4))
    return sg::refuse(me, "a buffer is not aligned to its entries");
  int dev = 0, sms = 0;
  if (const char* why = sg::current_device(&dev, &sms)) return sg::refuse(me, why);
  const Batch b = batch_of(sms, type, t, tokens, kv_heads, group, head_dim);
  if (!workspace || workspace_bytes < b.bytes)
    return sg::refuse(me, "the workspace is smaller than strasgpt_k_attn_shared_workspace says");
  if (!sg::aligned(workspace, 16)) return sg::refuse(me, "workspace must be 16-byte aligned");
  for (const void* p : {q, k_prefix, v_prefix, (const void*)prefix, k_cache, v_cache,
                        (const void*)rows, (const void*)first, (const void*)att,
                        (const void*)workspace})
    if (p)
      if (const char* why = sg::not_on_device(p, dev)) return sg::refuse(me, why);
  TreeArgs a = {};
  a.q = q; a.k = k_prefix; a.v = v_prefix; a.att = att;
  a.ldq = ldq; a.ldo = ldo;
  a.t = tokens; a.kh = kv_heads; a.group = group; a.ctx = prefix_ctx;
  a.cached = prefix;
  a.splits = b.splits;
  a.part = (float*)workspace;
  a.ml = (float2*)(a.part + b.parts * head_dim);
  sg::BatchArgs own = {};
  static_cast<TreeArgs&>(own) = a;
  own.k = k_cache; own.v = v_cache; own.ctx = ctx;
  own.requests = requests; own.most = t; own.first = first; own.rows = rows;
  own.stride = request_stride;
  own.ctas = b.ctas;
  own.split0 = b.splits;
  own.where = (int2*)((char*)workspace + b.where);
  const cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (type == STRASGPT_F32)
    e = head_dim == 128  ? launch_shared<float, 128>(a, own, dev, s)
        : head_dim == 64 ? launch_shared<float, 64>(a, own, dev, s)
                         : launch_shared<float, 32>(a, own, dev, s);
  else
    e = head_dim == 128  ? launch_shared<uint16_t, 128>(a, own, dev, s)
        : head_dim == 64 ? launch_shared<uint16_t, 64>(a, own, dev, s)
                         : launch_shared<uint16_t, 32>(a, own, dev, s);
  if (e != cudaSuccess) return sg::refuse_cuda(me, "launch", e);
  return 0;
}

}  // extern "C"
