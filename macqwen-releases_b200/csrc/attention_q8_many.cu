// attention_q8_many.cu -- causal attention over the paged 8-bit KV cache for
// sequences with many query rows (multi-token verify, prefill chunks), on
// tcgen05.  The arithmetic: attention_q8.cuh.
//
// A tile is 128 (row, head) pairs of one sequence and kv head (MMA M); a unit
// of work is a tile times 64 tokens.  k_q8_tiles lists the tiles with the
// units that causality leaves them; the units of all tiles, laid end to end,
// are dealt to persistent CTAs in equal contiguous ranges, so neither ragged
// lengths nor the causal triangle load one SM more than another.  Tiles that
// a range cuts are joined by k_q8_join.
//
// Per unit, S = Q K^T (M128 N64, K = D) and O += P V (M128 N = D, K = 64, for
// each of the two terms of P) run on the tensor cores with Q and P as TMEM
// operands, S and O as TMEM accumulators: 3 D * 128 * 64 multiply-adds where
// the formula has 2, at least 1,536 clocks a unit at D 256.
// Roles:
//   softmax     a row a thread (at D 256 two threads, 32 tokens each, which
//               exchange their maxima through shared memory): S from TMEM,
//               running reference and sum, P back to TMEM; Q in and the
//               result out of TMEM, through a shared-memory stage that turns
//               row-a-thread into coalesced 64-byte pieces;
//   one warp    issues the MMAs; another looks the units' scales up;
//   codes       read K and V codes (16 bytes a thread) one unit ahead in
//               registers, widen them to bfloat16 and store them to shared
//               memory as 128B-swizzled tiles, [D / 64][64 tokens][128 bytes]:
//               K-major for K, MN-major for V.
// The warpgroups trade registers (setmaxnreg): a softmax thread holds its part
// of a row of S, the issuer next to nothing.
// Widening in the kernel reads a byte a value from L2 where a widened copy
// would write and re-read two.
// TMEM columns at D 256: O 0-255, Q 256-383, S 384-447, P 448-511, so the next
// unit's Q K^T runs while this one's P is made.  At D 64 and 128 P takes S's
// columns and a CTA needs 256 of the 512: two CTAs share an SM and fill each
// other's waits.
// Measured: a 5,000-token prefill chunk (16/2 heads, D 256, 205 GFLOP) 368 us,
// 0.56 PFLOP/s, about 4,000 clocks a unit; at D 128 290 us and at D 64 235 us of
// half and a quarter of the work (these spill at 80 registers).  What bounds it now is the chain
// softmax -> P V and the issue slots that widening takes beside it (IPC 2.0);
// the MMAs alone take about 1,700 clocks a unit (N 64 and two terms of P).
// Every wait is bounded: a timeout sets the device error word and marks the
// CTA dead, whereupon every role leaves its loop.  The join then finds parts that
// were not written, but no descriptor that leads outside its arrays (cut_fits).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attention_q8.cuh"
#include "moe_kernels.cuh"
#include "umma.cuh"

namespace fnmoe {

namespace {

constexpr int kTile = 128;
constexpr int kInfo = 8;  // units whose scales are kept
constexpr uint32_t kSpin = 1u << 22;

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

template <int D>
struct Many {
  static constexpr bool kShared = D < 256;  // P takes S's columns
  static constexpr int kCtas = D < 256 ? 2 : 1;  // per SM
  static constexpr int kHalves = D < 256 ? 1 : 2;  // softmax threads a row
  static constexpr int kSoftWarps = 4 * kHalves;
  static constexpr int kMmaWarp = kSoftWarps;       // then the scales' warp, and two that fill the warpgroup
  static constexpr int kConvWarp0 = kMmaWarp + 4;
  static constexpr int kConvWarps = D < 256 ? 4 : 8;
  static constexpr int kThreads = 32 * (kConvWarp0 + kConvWarps);
  // Registers a thread: at launch 640 x 96 or 384 x 80; the shares add up to as many.
  static constexpr int kRegLaunch = D < 256 ? 80 : 96;
  static constexpr int kRegSoftmax = 136, kRegIssue = D < 256 ? 40 : 80, kRegConv = 64;
  static_assert(kHalves * kRegSoftmax + kRegIssue + kConvWarps / 4 * kRegConv <= kThreads / 128 * kRegLaunch, "registers");
  static constexpr int kSlots = 3;               // tiles of K and of V in shared memory
  static constexpr int kSlotBytes = 64 * D * 2;
  static constexpr int kCols = D < 256 ? 256 : 512;
  static constexpr int kColQ = D;
  static constexpr int kColS = D < 256 ? 192 : 384;
  static constexpr int kColP = D < 256 ? 192 : 448;
  // barriers
  static constexpr int kKFull = 0, kKEmpty = kKFull + kSlots, kVFull = kKEmpty + kSlots, kVEmpty = kVFull + kSlots,
                       kSFull = kVEmpty + kSlots, kSEmpty = kSFull + 1, kPFull = kSEmpty + 1, kPEmpty = kPFull + 1,
                       kQFull = kPEmpty + 1, kPair = kQFull + 1, kInfoFull = kPair + 4, kBars = kInfoFull + kInfo;
  static constexpr int kOffV = kSlots * kSlotBytes;
  static constexpr int kOffInfo = 2 * kSlots * kSlotBytes;  // float4 [kInfo][4]
  static constexpr int kOffMax = kOffInfo + kInfo * 64;      // float [2][2][128]: the halves' maxima, sums
  static constexpr int kOffStage = kOffMax + 2048;           // 32 rows x 64 bytes a softmax warp
  static constexpr int kOffBar = kOffStage + 2048 * kSoftWarps;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;      // TMEM base, dead flag
  static constexpr int kSmem = kOffMisc + 16 + 1024;        // + slack for the 1024-byte alignment of the tiles
  static constexpr int kMax = 148 * kCtas;
};
static_assert(Many<256>::kSmem <= 227 * 1024, "shared memory");
static_assert(2 * Many<128>::kSmem <= 227 * 1024, "shared memory of two CTAs");

// kind::f16, bfloat16 A and B, float32 D, M 128.
constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTile >> 4) << 24);
}
// Descriptor of a 128B-swizzled MN-major tile: 64-value groups of the MN
// dimension 8192 bytes apart (LBO), 8-token groups 1024 bytes apart (SBO).
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// D[tmem] (+)= A[tmem] B[smem].
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t s, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(s), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
// Bounded wait on `bar` for the phase of parity `parity`; false when it gives
// up or the CTA is dead.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *dead, uint32_t *err) {
  uint32_t spins = 0;
  while (!mbar_try_wait_u32(bar, parity)) {
    if (*dead) return false;
    if (++spins >= kSpin) {
      *dead = 1u;
      set_error(err, kErrTimeout);
      return false;
    }
  }
  return true;
}

// ---- tiles ------------------------------------------------------------------

__device__ __forceinline__ int tiles_of(const Q8View &p, int b) {
  const int rows = rows_of(p, b).y * p.gq;
  return rows > p.few_rows ? (rows + kTile - 1) / kTile : 0;
}

// Beginning and ending a tile costs about as much as kCost units (queries in,
// results out, the pipeline's start), which the ranges count: a tile and kv
// head of n units weighs n + kCost, and its real units are the last n of
// those.  (Prefill chunk of 5,000 tokens: weight 3 435 us, 4 406, 6 387, 8 388.)
constexpr int kCost = 6;

constexpr int kScanThreads = 1024;

// Inclusive sum over the CTA's threads plus `carry`, which becomes the total.
__device__ __forceinline__ long long scan1(long long v, long long &carry, long long *red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xFFFFFFFFu, v, off);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = red[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xFFFFFFFFu, w, off);
      if (lane >= off) w += o;
    }
    red[lane] = w;
  }
  __syncthreads();
  const long long before = warp > 0 ? red[warp - 1] : 0;
  const long long out = carry + before + v;
  carry += red[31];
  return out;
}

// One CTA: the tiles of all sequences and the units before each.
__global__ void __launch_bounds__(kScanThreads) k_q8_tiles(Q8View p) {
  __shared__ long long red[32];
  long long carry = 0;
  pdl_wait();
  pdl_trigger();
  for (int b0 = 0; b0 < p.B; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    const int n = b < p.B ? tiles_of(p, b) : 0;
    const long long s = scan1(n, carry, red);
    if (b < p.B) p.seq_tile[b] = static_cast<int>(s - n);
  }
  // Ascending cu_q never gives more than max_tiles.
  const int tiles = static_cast<int>(min(carry, static_cast<long long>(p.max_tiles)));
  if (threadIdx.x == 0) p.seq_tile[p.B] = tiles;
  __syncthreads();
  carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += kScanThreads) {
    const int t = t0 + threadIdx.x;
    long long units = 0;
    if (t < tiles) {
      int lo = 0, hi = p.B;  // the last sequence whose tiles begin at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.seq_tile[mid] <= t) lo = mid; else hi = mid;
      }
      const int mt = t - p.seq_tile[lo];
      const int n = rows_of(p, lo).y, rows = n * p.gq;
      const int last = (min((mt + 1) * kTile, rows) - 1) / p.gq;  // the tile's last query
      const int seen = max(0, min(p.ctx[lo] - n + last + 1, p.width * p.page));
      const int steps = (seen + kUnit - 1) / kUnit;
      p.tiles[t] = make_int4(lo, mt, steps, 0);
      units = steps > 0 ? static_cast<long long>(steps + kCost) * p.Hkv : 0;
    }
    const long long s = scan1(units, carry, red);
    if (t < tiles) p.tprefix[t] = s - units;
  }
  if (threadIdx.x == 0) p.tprefix[tiles] = carry;
  // No cut, until the CTA that makes one says so.  (Not by segment: k_q8_many does this.)
  if (p.tby_seg)
    for (int i = threadIdx.x; i < p.max_tiles * p.Hkv; i += kScanThreads) p.tcuts[i] = make_int4(-1, 0, 0, 0);
}

// The last of `tiles` tiles that begins at or before `unit`; a whole warp.
__device__ __forceinline__ int find_tile(const Q8View &p, int tiles, long long unit) {
  int lo = 0, hi = tiles;
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int t = lo + lane * step;
    const unsigned m = __ballot_sync(0xFFFFFFFFu, t < hi && p.tprefix[min(t, tiles)] <= unit);
    const int k = 31 - __clz(m);  // lane 0 always holds
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// A piece of work: units [u0, u0 + n) of a tile and kv head h.
struct Piece {
  int b, mt, h, u0, n, steps;
  bool first;  // of the CTA's range
};
struct Walk {
  long long cur, end, off, first;
  int tile;
};
__device__ __forceinline__ bool next_piece(const Q8View &p, Walk &w, Piece &q) {
  while (w.cur < w.end) {
    int4 t = p.tiles[w.tile];
    long long seg = t.z > 0 ? t.z + kCost : 0;
    while (w.off >= seg * p.Hkv) {
      w.off -= seg * p.Hkv;
      t = p.tiles[++w.tile];
      seg = t.z > 0 ? t.z + kCost : 0;
    }
    q.b = t.x;
    q.mt = t.y;
    q.steps = t.z;
    q.h = w.off <= 0xFFFFFFFFll ? static_cast<uint32_t>(w.off) / static_cast<uint32_t>(seg) : static_cast<int>(w.off / seg);
    const int v0 = static_cast<int>(w.off - q.h * seg);
    const int n = static_cast<int>(min(seg - v0, w.end - w.cur));
    q.u0 = max(v0 - kCost, 0);
    q.n = max(v0 + n - kCost, 0) - q.u0;
    q.first = w.cur == w.first;
    w.cur += n;
    w.off += n;
    if (q.n > 0) return true;  // else the range ends in the tile's overhead
  }
  return false;
}

// 16 codes to 16 bfloat16.
template <bool E4M3>
__device__ __forceinline__ void widen16(uint4 c, uint4 &lo, uint4 &hi) {
  lo = make_uint4(widen2<E4M3, 0>(c.x), widen2<E4M3, 1>(c.x), widen2<E4M3, 0>(c.y), widen2<E4M3, 1>(c.y));
  hi = make_uint4(widen2<E4M3, 0>(c.z), widen2<E4M3, 1>(c.z), widen2<E4M3, 0>(c.w), widen2<E4M3, 1>(c.w));
}

// Tiles that see no token: their rows are zero.
template <int D>
__device__ __forceinline__ void zero_tiles(const Q8View &p, int tiles) {
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int4 ti = p.tiles[t];
    if (ti.z != 0) continue;
    const int2 qr = rows_of(p, ti.x);
    const int r0 = ti.y * kTile, nr = min(kTile, qr.y * p.gq - r0);
    for (int i = threadIdx.x; i < nr * p.Hkv * (D / 8); i += blockDim.x) {
      const int d = i % (D / 8), rh = i / (D / 8);
      const int r = r0 + rh % nr, h = rh / nr;
      const int qi = r / p.gq, head = h * p.gq + r - qi * p.gq;
      *reinterpret_cast<uint4 *>(p.out + (static_cast<size_t>(qr.x + qi) * p.Hq + head) * D + 8 * d) = make_uint4(0, 0, 0, 0);
    }
  }
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(Many<D>::kThreads, Many<D>::kCtas) k_q8_many(Q8View p, uint32_t *err) {
  using M = Many<D>;
  extern __shared__ uint8_t many_raw[];
  pdl_wait();
  pdl_trigger();
  const uint32_t raw0 = smem_u32(many_raw);
  const uint32_t sbase = (raw0 + 1023u) & ~1023u;
  uint8_t *sm = many_raw + (sbase - raw0);
  const uint32_t bars = sbase + M::kOffBar;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + M::kOffMisc);
  volatile uint32_t *dead = reinterpret_cast<volatile uint32_t *>(sm + M::kOffMisc + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int tiles = p.seq_tile[p.B];
  const long long total = p.tprefix[tiles];
  const Ranges ranges(total, gridDim.x);
  Walk w;
  w.cur = w.first = ranges.begin(blockIdx.x);
  w.end = ranges.begin(blockIdx.x + 1);
  if (w.cur >= w.end) {
    if (tid == 0 && !p.tby_seg) p.tcuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
    zero_tiles<D>(p, tiles);
    return;
  }
  w.tile = find_tile(p, tiles, w.cur);
  w.off = w.cur - p.tprefix[w.tile];

  if (tid == 0) {
    for (int i = 0; i < M::kBars; ++i) {
      uint32_t count = 1;
      if ((i >= M::kKFull && i < M::kKFull + M::kSlots) || (i >= M::kVFull && i < M::kVFull + M::kSlots)) count = M::kConvWarps;
      if (i == M::kSEmpty || i == M::kPFull || i == M::kQFull) count = M::kSoftWarps;
      if (i >= M::kPair && i < M::kPair + 4) count = 2;
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bars + 8 * i), "r"(count));
    }
    *dead = 0u;
    mbar_init_fence();
    if (!p.tby_seg) p.tcuts[blockIdx.x] = make_int4(-1, 0, 0, 0);  // until the first piece shows a cut
  }
  if (warp == M::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(static_cast<uint32_t>(M::kCols)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto bar = [&](int i) { return bars + 8 * i; };
  Piece q;

  if (warp < M::kSoftWarps) {
    // ---------------- softmax: a row and kTok tokens of each unit a thread ----------------
    reg_inc<M::kRegSoftmax>();
    constexpr int kTok = kUnit / M::kHalves;  // tokens of this thread
    constexpr int kDims = D / M::kHalves;     // dims of Q and O that it moves
    const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    const uint32_t stage = sbase + M::kOffStage + 2048 * warp;
    // This thread's 16-byte chunk c of its own row in the stage, and the chunk
    // of row 8 e + lane / 4 that it moves to or from global memory.
    auto own = [&](int c) { return stage + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4); };
    auto other = [&](int e) {
      const int r = 8 * e + (lane >> 2);
      return stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4);
    };
    // The other half's value for this row; buffers alternate, so that one is
    // rewritten only after both halves have read it.
    uint32_t exchanges = 0;
    bool live = true;
    auto swap = [&](float mine) {
      volatile float *sx = reinterpret_cast<volatile float *>(sm + M::kOffMax) + (exchanges & 1u) * 256;
      sx[half * 128 + row] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(M::kPair + quarter));
      live = __all_sync(0xFFFFFFFFu, bar_wait(bar(M::kPair + quarter), exchanges & 1u, dead, err));
      ++exchanges;
      return sx[(half ^ 1) * 128 + row];
    };
    uint32_t i = 0;  // units so far
    while (live && next_piece(p, w, q)) {
      const int2 qr = rows_of(p, q.b);
      const int rows = qr.y * p.gq;
      const int r = q.mt * kTile + row;
      const bool valid = r < rows;
      const int qi = valid ? r / p.gq : 0, head = q.h * p.gq + (valid ? r - qi * p.gq : 0);
      // Last position the row sees; rows past the end are left unmasked (and unwritten).
      const int lim = valid ? p.ctx[q.b] - qr.y + qi : 0x7FFFFFFF;
      const int lim_min = __reduce_min_sync(0xFFFFFFFFu, lim);
      const bool idle = !__any_sync(0xFFFFFFFFu, valid);
      if (tid == 0) {
        const bool cut = q.first && q.u0 > 0;
        const long long a = w.cur - (kCost + q.u0 + q.n);  // the segment's first unit, of a piece that does not end it
        const int4 c4 = cut ? cut_of(ranges, q.b, q.h, q.mt, a, a + kCost, a + kCost + q.steps - 1, blockIdx.x)
                            : make_int4(-1, 0, 0, 0);
        if (p.tby_seg) {  // the first cut in a segment, or the CTA that does it all
          if (c4.x >= 0 || (q.u0 == 0 && q.n == q.steps))
            p.tcuts[static_cast<size_t>(w.tile) * p.Hkv + q.h] = make_int4(c4.x, blockIdx.x - 1, c4.z, c4.w);
        } else if (cut) {
          p.tcuts[blockIdx.x] = c4;
        }
      }
      // Rows of the warp that this thread moves: row 8 e + lane / 4.
      long long q_at[4], o_at[4];
      {
        const long long qa = valid ? static_cast<long long>(static_cast<uint64_t>(qr.x + qi) * p.q_stride + static_cast<uint64_t>(head) * D) : -1;
        const long long oa = (static_cast<long long>(qr.x + qi) * p.Hq + head) * D;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q_at[e] = __shfl_sync(0xFFFFFFFFu, qa, 8 * e + (lane >> 2));
          o_at[e] = __shfl_sync(0xFFFFFFFFu, oa, 8 * e + (lane >> 2));
          if (q_at[e] < 0) o_at[e] = -1;
        }
      }
      {  // Q into TMEM; the last piece's products are done (its sums were read)
        const int c0 = half * kDims + 8 * (lane & 3);
        uint4 x[kDims / 32][4];
#pragma unroll
        for (int c = 0; c < kDims / 32; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[c][e] = q_at[e] >= 0 ? __ldcg(reinterpret_cast<const uint4 *>(p.q + q_at[e] + c0 + 32 * c)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < kDims / 32; ++c) {
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 4; ++e) sts128(other(e), x[c][e]);
          __syncwarp();
          uint32_t v[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 y = lds128(own(e));
            v[4 * e] = y.x;
            v[4 * e + 1] = y.y;
            v[4 * e + 2] = y.z;
            v[4 * e + 3] = y.w;
          }
          tmem_st16(lanes + M::kColQ + (half * kDims) / 2 + 16 * c, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(M::kQFull));
      }
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < q.n; ++j, ++i) {
        live = bar_wait(bar(M::kInfoFull + i % kInfo), (i / kInfo) & 1u, dead, err) &&
               bar_wait(bar(M::kSFull), i & 1u, dead, err);
        live = __all_sync(0xFFFFFFFFu, live);
        if (!live) break;
        tc_fence_after();
        float s[kTok];
        if (!idle) {
#pragma unroll
          for (int c = 0; c < kTok / 32; ++c)
            tmem_ld32_nowait(lanes + M::kColS + half * kTok + 32 * c, reinterpret_cast<uint32_t *>(s + 32 * c));
          tmem_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        if (!M::kShared && lane == 0) mbar_arrive(bar(M::kSEmpty));
        if (!idle) {
          const int t0 = (q.u0 + j) * kUnit + half * kTok;
          if (t0 + kTok - 1 > lim_min) {
#pragma unroll
            for (int e = 0; e < kTok; ++e) s[e] = t0 + e <= lim ? s[e] : -INFINITY;
          }
          const float4 *info = reinterpret_cast<const float4 *>(sm + M::kOffInfo) + (i % kInfo) * 4 + half * (kTok / 16);
          float4 f[kTok / 16];
          float tm = -INFINITY;
#pragma unroll
          for (int g = 0; g < kTok / 16; ++g) {
            f[g] = info[g];  // scale * log2 e * ks, log2 vs', 1 / vs', vs / vs'
            float a = s[16 * g], b = s[16 * g + 1];
#pragma unroll
            for (int e = 2; e < 16; e += 2) {
              a = fmaxf(a, s[16 * g + e]);
              b = fmaxf(b, s[16 * g + e + 1]);
            }
            tm = fmaxf(tm, __fmaf_rn(fmaxf(a, b), f[g].x, f[g].y));
          }
          if (M::kHalves == 2) {
            const float o = swap(tm);
            if (!live) break;
            tm = fmaxf(tm, o);
          }
          if (__any_sync(0xFFFFFFFFu, tm > m + kLazy)) {
            const float mn = fmaxf(m, tm);
            const float al = mn == -INFINITY ? 1.0f : ex2(m - mn);
            if (mn != -INFINITY) l = times_ex2(l, m - mn);
            m = mn;
            if (j > 0) {
              live = __all_sync(0xFFFFFFFFu, bar_wait(bar(M::kPEmpty), (i & 1u) ^ 1u, dead, err));
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < kDims / 32; ++c) {
                uint32_t v[32];
                tmem_ld32_nowait(lanes + half * kDims + 32 * c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * al);
                tmem_st32(lanes + half * kDims + 32 * c, v);
              }
              tmem_wait_st();
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
          for (int h2 = 0; h2 < kTok / 32; ++h2) {
            uint32_t hi[16], lo[16];
            auto weigh = [&](auto folds) {
#pragma unroll
              for (int g2 = 0; g2 < 2; ++g2) {
                const int g = 2 * h2 + g2;
                const float2 mul = make_float2(f[g].x, f[g].x), add = make_float2(f[g].y - ref, f[g].y - ref);
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const float2 x = fma2(make_float2(s[16 * g + e], s[16 * g + e + 1]), mul, add);
                  float2 u = make_float2(ex2(x.x), ex2(x.y));
                  sum = add2(sum, u);
                  if constexpr (decltype(folds)::value) u = make_float2(u.x * f[g].w, u.y * f[g].w);
                  // hi: the upper 16 bits of each; lo: what is left, rounded
                  const uint32_t a0 = __float_as_uint(u.x), a1 = __float_as_uint(u.y);
                  hi[8 * g2 + e / 2] = prmt(a0, a1, 0x7632u);
                  const float2 left = add2(u, make_float2(__uint_as_float((a0 & 0xFFFF0000u) ^ 0x80000000u),
                                                          __uint_as_float((a1 & 0xFFFF0000u) ^ 0x80000000u)));
                  lo[8 * g2 + e / 2] = pack_bf16x2(left.x, left.y);
                }
                l = __fmaf_rn(sum.x + sum.y, f[g].z, l);
              }
            };
            if (f[2 * h2].w == 1.0f && f[2 * h2 + 1].w == 1.0f)  // alike in all threads of the warp
              weigh(std::false_type{});
            else
              weigh(std::true_type{});
            if (h2 == 0) {  // P may be written once the last unit's P V is done
              live = live && bar_wait(bar(M::kPEmpty), (i & 1u) ^ 1u, dead, err);
              live = __all_sync(0xFFFFFFFFu, live);
              if (!live) break;
              tc_fence_after();
            }
            tmem_st16(lanes + M::kColP + 16 * (half + h2), hi);
            tmem_st16(lanes + M::kColP + 32 + 16 * (half + h2), lo);
          }
          if (!live) break;
          tmem_wait_st();
        } else {
          live = __all_sync(0xFFFFFFFFu, bar_wait(bar(M::kPEmpty), (i & 1u) ^ 1u, dead, err));
          if (!live) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(M::kPFull));
      }
      if (!live) break;
      // ---- the tile's (or the piece's) sums ----
      live = __all_sync(0xFFFFFFFFu, bar_wait(bar(M::kPEmpty), (i - 1) & 1u, dead, err));
      if (!live) break;
      tc_fence_after();
      if (!idle) {
        if (M::kHalves == 2) {
          const float o = swap(l);
          if (!live) break;
          l += o;
        }
        const bool whole = q.u0 == 0 && q.n == q.steps;
        const float inv = l > 0.0f ? __frcp_rn(l) : 0.0f;
        const int slot = 2 * blockIdx.x + (q.first ? 0 : 1);
        // cut tiles: float4 d of row r at [d][r], so that a warp's stores are contiguous
        float4 *part = reinterpret_cast<float4 *>(p.tpart) + (static_cast<size_t>(slot) * (D / 4) + half * (kDims / 4)) * kTile + row;
        uint32_t vv[2][32];
        tmem_ld32_nowait(lanes + half * kDims, vv[0]);
#pragma unroll
        for (int c = 0; c < kDims / 32; ++c) {
          uint32_t (&v)[32] = vv[c & 1];
          __syncwarp();
          tmem_wait_ld();
          if (c + 1 < kDims / 32) tmem_ld32_nowait(lanes + half * kDims + 32 * (c + 1), vv[(c + 1) & 1]);
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                o[k] = pack_bf16x2(__uint_as_float(v[8 * e + 2 * k]) * inv, __uint_as_float(v[8 * e + 2 * k + 1]) * inv);
              sts128(own(e), make_uint4(o[0], o[1], o[2], o[3]));
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (o_at[e] >= 0)
                *reinterpret_cast<uint4 *>(p.out + o_at[e] + half * kDims + 32 * c + 8 * (lane & 3)) = lds128(other(e));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              part[(8 * c + e) * kTile] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                                      __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
          }
        }
        if (!whole && half == 0) p.tpart_ml[slot * kTile + row] = make_float2(m, l);
      }
      tc_fence_before();  // the next piece's products overwrite what was read
      __syncwarp();
    }
  } else if (warp < M::kConvWarp0) {
    // ---------------- MMA issuer ----------------
    reg_dec<M::kRegIssue>();
    if (warp == M::kMmaWarp) {
      // The whole warp walks the units (so that descriptors stay in uniform
      // registers); one elected lane issues.
      uint32_t nk = 0, nv = 0, pieces = 0;  // units whose Q K^T / P V were issued
      uint32_t kslot = 0, kph = 0, vslot = 0, vph = 0;
      bool live = true;
      const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
      auto wait = [&](int i, uint32_t parity) { return __all_sync(0xFFFFFFFFu, bar_wait(bar(i), parity, dead, err)) != 0; };
      auto pv = [&](bool accumulate) {
        live = wait(M::kVFull + vslot, vph) && wait(M::kPFull, nv & 1u);
        if (!live) return;
        tc_fence_after();
        const uint64_t vd = sw128_mn_desc(sbase + M::kOffV + vslot * M::kSlotBytes);
        if (elect_one()) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ts(tm, tm + M::kColP + 32 * half + 8 * kk, vd + 128 * kk, idesc(D, true),
                      accumulate || half + kk > 0 ? 1u : 0u);
          umma_commit(bar(M::kVEmpty + vslot));
          umma_commit(bar(M::kPEmpty));
        }
        __syncwarp();
        ++nv;
        if (++vslot == M::kSlots) {
          vslot = 0;
          vph ^= 1u;
        }
      };
      while (live && next_piece(p, w, q)) {
        const int n = __shfl_sync(0xFFFFFFFFu, q.n, 0);
        live = wait(M::kQFull, pieces & 1u);
        ++pieces;
        for (int j = 0; live && j < n; ++j) {
          // S free: read by the softmax, or (shared columns) P consumed by P V
          live = wait(M::kShared ? M::kPEmpty : M::kSEmpty, (nk & 1u) ^ 1u) && wait(M::kKFull + kslot, kph);
          if (!live) break;
          tc_fence_after();
          const uint64_t kd = sw128_desc(sbase + kslot * M::kSlotBytes);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_ts(tm + M::kColS, tm + M::kColQ + 8 * kk, kd + 512 * (kk / 4) + 2 * (kk % 4), idesc(64, false),
                      kk > 0 ? 1u : 0u);
            umma_commit(bar(M::kKEmpty + kslot));
            umma_commit(bar(M::kSFull));
          }
          __syncwarp();
          ++nk;
          if (++kslot == M::kSlots) {
            kslot = 0;
            kph ^= 1u;
          }
          if (M::kShared)
            pv(j > 0);
          else if (j > 0)
            pv(j > 1);
        }
        if (!M::kShared && live) pv(n > 1);
      }
      // Products may still be under way when another role gave up: they end (or a
      // bounded wait does) before the TMEM that they write is freed.
      auto settle = [&](int i, uint32_t units) {
        if (units > 0)
          for (uint32_t spins = 0; spins < kSpin && !mbar_try_wait_u32(bar(i), (units - 1) & 1u); ++spins) {
          }
      };
      settle(M::kSFull, nk);
      settle(M::kPEmpty, nv);
    } else if (warp == M::kMmaWarp + 1) {
      // ---------------- the units' scales: a lane for each granule of 16 tokens ----------------
      uint32_t i = 0;
      bool live = true;
      while (live && next_piece(p, w, q)) {
        const int ctx = tokens_of(p, q.b), bpp = p.page >> p.block_shift;
        const int32_t *trow = p.table + static_cast<size_t>(q.b) * p.width;
        float v_top = 0.0f;  // the largest value scale of the piece so far
        for (int u = q.u0; live && u < q.u0 + q.n; ++u, ++i) {
          const uint32_t slot = i % M::kSlots, ph = (i / M::kSlots) & 1u;
          const int t = u * kUnit + 16 * (lane & 3);
          float mul = 1e-37f, add = -INFINITY, inv = 0.0f, fold = 1.0f;  // a granule without a token or page weighs nothing
          float v = -1.0f;
          if (t < ctx) {
            const int c = page_col(p, t), pg = trow[c];
            if (static_cast<uint32_t>(pg) < static_cast<uint32_t>(p.pages)) {
              const size_t at = (static_cast<size_t>(pg) * bpp + ((t - c * p.page) >> p.block_shift)) * p.Hkv + q.h;
              v = fmaxf(__ldcg(p.vs + at), 0.0f);
              mul = fmaxf(p.scale * kLog2e * __ldcg(p.ks + at), 1e-37f);
            }
          }
          // bits of numbers that are not negative order as the numbers do
          v_top = fmaxf(v_top, __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fmaxf(v, 0.0f)))));
          if (v >= 0.0f) {
            const float v_least = fmaxf(v_top * kScaleSpan, kScaleLeast), v_scale = fmaxf(v, v_least);
            add = lg2(v_scale);
            inv = rcp(v_scale);
            if (v < v_least) fold = v * inv;
          }
          // as far ahead as K itself may be, so that the kept units are not overrun
          live = __all_sync(0xFFFFFFFFu, bar_wait(bar(M::kKEmpty + slot), ph ^ 1u, dead, err));
          if (!live) break;
          if (lane < 4) reinterpret_cast<float4 *>(sm + M::kOffInfo)[(i % kInfo) * 4 + lane] = make_float4(mul, add, inv, fold);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(M::kInfoFull + i % kInfo));
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- codes to shared memory ----------------
    if constexpr (M::kRegConv < M::kRegLaunch) reg_dec<M::kRegConv>();
    constexpr int kPer = D / 16;                          // 16-code chunks of a row
    constexpr int kRowsPass = 32 * M::kConvWarps / kPer;  // rows of a pass: 16 or 32
    constexpr int kPasses = kUnit / kRowsPass;
    // Four lanes take a 64-value group of one row, the next four the same group
    // of the next row: their eight 16-byte stores hit all eight bank groups.
    constexpr int kGroups = D / 64;
    const int ct = tid - 32 * M::kConvWarp0;
    const int grp = (ct >> 3) % kGroups, c4 = ct & 3;
    const int row0 = 2 * (ct / (8 * kGroups)) + ((ct >> 2) & 1);
    const uint32_t soff = grp * 8192 + row0 * 128 + (((2 * c4) ^ (row0 & 7)) << 4);  // second half: ^ 16
    const uint32_t row_bytes = static_cast<uint32_t>(p.Hkv) * D;
    // 16-token granule g of a unit lies in one page: lane g looks its first slot
    // up, a unit ahead, and the warp shuffles it (a warp's rows of a pass are of
    // one granule).
    const int row16 = row0 & 15, g0 = row0 >> 4;
    constexpr int kGranules = kRowsPass / 16;  // from one pass to the next
    uint32_t i = 0;
    bool live = true;
    while (live && next_piece(p, w, q)) {
      const int ctx = tokens_of(p, q.b);
      const int32_t *trow = p.table + static_cast<size_t>(q.b) * p.width;
      const int last = q.u0 + q.n;
      const size_t off = static_cast<size_t>(row16) * row_bytes + static_cast<size_t>(q.h) * D + 64 * grp + 16 * c4;
      const uint8_t *kbase = p.kc + off, *vbase = p.vc + off;
      int slot_next = -1;  // lane g < 4: granule g's first slot, -1 without a token or page
      int pg_after = -1, in_after = 0;  // of the unit after that: its page, still on its way
      auto look_up = [&](int u) {
        const int t = u * kUnit + 16 * (lane & 3), c = page_col(p, t);
        in_after = t - c * p.page;
        pg_after = t < ctx ? trow[c] : -1;
      };
      auto advance = [&]() {
        slot_next = static_cast<uint32_t>(pg_after) < static_cast<uint32_t>(p.pages) ? pg_after * p.page + in_after : -1;
      };
      uint4 ck[kPasses], cv[kPasses];
      auto fetch = [&](const uint8_t *codes, uint4 (&c)[kPasses]) {
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int s0 = __shfl_sync(0xFFFFFFFFu, slot_next, g0 + k * kGranules);
          c[k] = ldg_stream(codes + static_cast<uint64_t>(static_cast<uint32_t>(max(s0, 0))) * row_bytes);
        }
      };
      // Passes of unit u whose token is past the context or has no page.  They
      // weigh nothing, but e4m3 codes can be NaN: those are stored as zeros
      // (when they are stored: touching them before would wait for the loads).
      auto missing = [&](int u) {
        uint32_t m = 0;
        if (E4M3 && (!__all_sync(0xFFFFFFFFu, slot_next >= 0) || (u + 1) * kUnit > ctx)) {
#pragma unroll
          for (int k = 0; k < kPasses; ++k) {
            const int s0 = __shfl_sync(0xFFFFFFFFu, slot_next, g0 + k * kGranules);
            if (s0 < 0 || u * kUnit + k * kRowsPass + row0 >= ctx) m |= 1u << k;
          }
        }
        return m;
      };
      auto store = [&](uint32_t tile, uint4 (&c)[kPasses], uint32_t zero) {
        if (E4M3 && __any_sync(0xFFFFFFFFu, zero != 0)) {
#pragma unroll
          for (int k = 0; k < kPasses; ++k)
            if ((zero >> k) & 1u) c[k] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          uint4 a, b;
          widen16<E4M3>(c[k], a, b);
          const uint32_t at = tile + soff + k * (kRowsPass * 128);
          sts128(at, a);
          sts128(at ^ 16u, b);
        }
      };
      look_up(q.u0);
      advance();
      fetch(kbase, ck);
      fetch(vbase, cv);
      uint32_t zero = missing(q.u0), zero_next = 0;
      look_up(q.u0 + 1);
      for (int u = q.u0; u < last; ++u, ++i) {
        const uint32_t slot = i % M::kSlots, ph = (i / M::kSlots) & 1u;
        advance();
        look_up(u + 2);
        live = bar_wait(bar(M::kKEmpty + slot), ph ^ 1u, dead, err);
        live = __all_sync(0xFFFFFFFFu, live);
        if (!live) break;
        store(sbase + slot * M::kSlotBytes, ck, zero);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(M::kKFull + slot));
        if (u + 1 < last) {
          fetch(kbase, ck);
          zero_next = missing(u + 1);
        }
        live = bar_wait(bar(M::kVEmpty + slot), ph ^ 1u, dead, err);
        live = __all_sync(0xFFFFFFFFu, live);
        if (!live) break;
        store(sbase + M::kOffV + slot * M::kSlotBytes, cv, zero);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(M::kVFull + slot));
        if (u + 1 < last) {
          fetch(vbase, cv);
        }
        zero = zero_next;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  zero_tiles<D>(p, tiles);
  if (warp == M::kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                 "r"(static_cast<uint32_t>(M::kCols)));
}

template <int D, bool E4M3>
cudaError_t launch(const Q8View &p, cudaStream_t s) {
  using M = Many<D>;
  static SmemLimit limit;
  cudaError_t e = limit.set(reinterpret_cast<const void *>(k_q8_many<D, E4M3>), M::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_q8_tiles, dim3(1), dim3(kScanThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_q8_many<D, E4M3>, dim3(M::kMax), dim3(M::kThreads), M::kSmem, s, p, device_error_word());
}

}  // namespace

int many_ctas(int head_dim) { return head_dim == 256 ? Many<256>::kMax : Many<128>::kMax; }

uint64_t many_tiles(const Q8View &p) {
  const uint64_t pairs = static_cast<uint64_t>(p.rows) * p.gq;
  // a full tile per 128 pairs, a partial one per sequence that can be here
  return pairs / kTile + std::min<uint64_t>(p.B, pairs / (p.few_rows + 1) + 1);
}

cudaError_t launch_many(const Q8View &p, int head_dim, bool e4m3, cudaStream_t s) {
  switch (head_dim) {
    case 64: return e4m3 ? launch<64, true>(p, s) : launch<64, false>(p, s);
    case 128: return e4m3 ? launch<128, true>(p, s) : launch<128, false>(p, s);
    default: return e4m3 ? launch<256, true>(p, s) : launch<256, false>(p, s);
  }
}

}  // namespace fnmoe
