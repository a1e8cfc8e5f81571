// attention_q8.cu -- causal attention over the paged 8-bit KV cache (sm_100a):
// the entry points and the kernels for sequences with few query rows (decode).
// The arithmetic: attention_q8.cuh; many rows: attention_q8_many.cu.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>
#include <type_traits>

#include "attention_q8.cuh"
#include "moe_kernels.cuh"
#include "paged_q8.cuh"
#include "umma.cuh"

namespace fnmoe {

namespace {

// ---- few rows per sequence --------------------------------------------------
//
// Bound by HBM (one byte a value, 2 * D * Hkv bytes a token).  Work is cut
// into units of 128 tokens of one (sequence, kv head, tile of 8 rows); the
// units of all sequences, laid end to end, are dealt to the CTAs in equal
// contiguous ranges, so ragged contexts load every SM alike.  A CTA's range
// covers whole segments, which it finishes, and at most two cut ones (its
// first and last), whose sums go to the workspace for k_q8_join.
//
// A warp takes 32 tokens at a time, as two tiles of 16 whose chains of
// dependent instructions overlap.  It fetches them for itself: TMA boxes of
// 16 or 32 tokens x 128 bytes (128-byte swizzle; 64 bytes at D 64) into shared
// memory of its own, the next step's K as soon as this one's scores are done, the next
// V when its products are; no warp waits for another inside a piece of work.
// (Loads by the lanes themselves, to registers or by cp.async, stayed at
// 3.5 TB/s whatever the occupancy.)
//   S^T = K Q^T   (M = 16 tokens, N = 8 rows): A fragments by ldmatrix
//     (QueryInt8, QueryE4M3);
//   O^T += V^T P^T (M = 16 dims, N = 8 rows, K = 16 tokens): lane (g, t)
//     takes 16 consecutive dims of tokens 2t, 2t+1, 2t+8, 2t+9 and pairs the
//     tokens' bytes with prmt.
// 16 tokens lie in one page and one scale block.
//
// Measured: 16 sequences of 1k-32k tokens (16/2 heads, D 256; 290 MB) 66 us with
// the join, 4.4 TB/s; 16 x 131,072 tokens 6.1 TB/s (94% of a measured copy) at D
// 256 and 128, 4.6 TB/s at D 64 (64-byte pieces; the kernel also spills).  The rest is a
// fixed 20 us: launch, finding the range, the first copies, joining warps and
// CTAs.

constexpr int kFewThreads = 128;
constexpr int kFewUnit = 128;  // 4 warps x 32 tokens
// Sequences of more (row, head) pairs a kv head go to the many-row kernel: each
// tile of 8 here reads and widens the cache again.  16 sequences of 1 to 8 rows
// of 8 heads: 8 90 us, 16 90, 24 99, 32 110.
constexpr int kFewRows = 16;
constexpr uint32_t kFewSpin = 1u << 22;  // mbarrier polls before a wait gives up

// A step's codes of K (or V): 32 rows of 128 bytes, chunk c of a row at
// c ^ (row & 7), for each 128-byte piece of D (the boxes' swizzle); at D 64, 32
// rows of 64 bytes, c at c ^ ((row >> 1) & 3).  Rows 16 and on are the second
// tile.  tile_offset: where chunk c of the first piece of a tile's row is.
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int row, int c) {
  return D == 64 ? row * 64 + ((c ^ ((row >> 1) & 3)) << 4) : row * 128 + ((c ^ (row & 7)) << 4);
}
// 2 st chunks on from one of a row's first two: the chunk's bits are
// exclusive-ored, and the next piece follows 4096 bytes later.
template <int D>
__device__ __forceinline__ uint32_t step_offset(uint32_t off, int st) {
  return (off ^ ((2 * (st & 3)) << 4)) + (st >> 2) * 4096;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The query rows as B operands in shared memory (fragment order, shared by the
// CTA's warps), and the scores of two tiles of 16 tokens at at[0], at[1].
// ldmatrix gives lane (g, t) the codes of tokens g and g + 8 at dims 32 s + 4 t
// .. + 3 and 32 s + 16 + 4 t .. + 3; put() stores this lane's share of 32-dim
// step s of its row (eight dims, as two words a, b of four: the raw bfloat16
// pairs); scale_of() is the power of two that a row's scores are to be
// multiplied by, from the bits of its largest magnitude.
//
// e4m3 codes and queries as float16: the codes are exact, one conversion for
// two; a row is scaled so that its largest element lies in [1, 2) (exact for
// elements within 2^-14 of it).
template <int D>
struct QueryE4M3 {
  static constexpr int kBytes = D / 16 * 256;
  static __device__ __forceinline__ uint32_t exponent(uint32_t peak) { return min(max(peak >> 7, 1u), 253u); }
  static __device__ __forceinline__ float scale_of(uint32_t peak) { return __uint_as_float(exponent(peak) << 23); }
  static __device__ __forceinline__ void put(uint2 *q, int s, uint2 a, uint2 b, uint32_t peak) {
    const float down = __uint_as_float((254u - exponent(peak)) << 23);
    auto pair = [&](uint32_t w) { return pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down); };
    const int lane = threadIdx.x & 31;
    q[2 * s * 32 + lane] = make_uint2(pair(a.x), pair(a.y));
    q[(2 * s + 1) * 32 + lane] = make_uint2(pair(b.x), pair(b.y));
  }
  static __device__ __forceinline__ void scores(const uint32_t (&at)[2], uint32_t q, float (&s)[2][4]) {
    const uint32_t off = tile_offset<D>(threadIdx.x & 15, (threadIdx.x >> 4) & 1);
    float c[2][2][4] = {};  // two chains a tile
#pragma unroll
    for (int st = 0; st < D / 32; ++st) {
      uint32_t w[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) ldsm_x4(at[u] + step_offset<D>(off, st), w[u]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 b = lds64(q + (2 * st + k) * 256);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t x0 = w[u][2 * k], x1 = w[u][2 * k + 1];
          const uint32_t a[4] = {e4m3_f16<0>(x0), e4m3_f16<0>(x1), e4m3_f16<1>(x0), e4m3_f16<1>(x1)};
          mma_16816(c[u][k], a, b.x, b.y);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][e] = __fadd_rn(c[u][0][e], c[u][1][e]);
  }
};

// int8 codes as they are, on the integer tensor cores: a row as the fixed
// point X = round(q 2^(21 - E)), E the exponent of its largest element, in
// three byte planes X = X0 + 2^8 X1 + 2^16 X2 (X2 signed); sums of code times
// plane stay below 2^24, exact in float32.  X is exact for elements within
// 2^-14 of the largest.
template <int D>
struct QueryInt8 {
  static constexpr int kBytes = 3 * (D / 32) * 256;
  static __device__ __forceinline__ uint32_t exponent(uint32_t peak) { return min(max(peak >> 7, 24u), 253u); }
  static __device__ __forceinline__ float scale_of(uint32_t peak) {  // NaN for a row with an infinity or NaN
    return (peak >> 7) == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((exponent(peak) - 21u) << 23);
  }
  static __device__ __forceinline__ void put(uint2 *q, int s, uint2 a, uint2 b, uint32_t peak) {
    const float up = __uint_as_float((275u - exponent(peak)) << 23);  // 2^(21 - E)
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
    uint32_t plane[3][2] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k)  // four dims: one word of each plane
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t v = w[2 * k + (t >> 1)];
        const int x = __float2int_rn(__uint_as_float(t & 1 ? v & 0xFFFF0000u : v << 16) * up);
#pragma unroll
        for (int p = 0; p < 3; ++p) plane[p][k] |= ((static_cast<uint32_t>(x) >> (8 * p)) & 0xFFu) << (8 * t);
      }
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int p = 0; p < 3; ++p) q[(p * (D / 32) + s) * 32 + lane] = make_uint2(plane[p][0], plane[p][1]);
  }
  static __device__ __forceinline__ void scores(const uint32_t (&at)[2], uint32_t q, float (&s)[2][4]) {
    const uint32_t off = tile_offset<D>(threadIdx.x & 15, (threadIdx.x >> 4) & 1);
    int c[2][3][4] = {};
#pragma unroll
    for (int st = 0; st < D / 32; ++st) {
      const uint2 b0 = lds64(q + st * 256), b1 = lds64(q + (D / 32 + st) * 256), b2 = lds64(q + (2 * (D / 32) + st) * 256);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t a[4];
        ldsm_x4(at[u] + step_offset<D>(off, st), a);
        mma_s8<false>(c[u][0], a[0], a[1], a[2], a[3], b0.x, b0.y);
        mma_s8<false>(c[u][1], a[0], a[1], a[2], a[3], b1.x, b1.y);
        mma_s8<true>(c[u][2], a[0], a[1], a[2], a[3], b2.x, b2.y);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[u][e] = __fmaf_rn(__int2float_rn(c[u][2][e]), 65536.0f,
                            __fmaf_rn(__int2float_rn(c[u][1][e]), 256.0f, __int2float_rn(c[u][0][e])));
  }
};

template <int D, bool E4M3>
struct Few {
  using Query = typename std::conditional<E4M3, QueryE4M3<D>, QueryInt8<D>>::type;
  static constexpr int kCtas = D == 256 ? 3 : D == 128 ? 4 : 6;  // per SM
  static constexpr int kTileBytes = 16 * D;                     // K (or V) codes of 16 tokens
  static constexpr int kWarpBytes = 4 * kTileBytes;             // two tiles of K, two of V
  static constexpr int kOffQ = 4 * kWarpBytes;                  // the warps' sums are joined in the first part
  static constexpr int kOffBar = kOffQ + Query::kBytes;         // per warp: K has arrived, V has arrived
  static constexpr int kSmem = kOffBar + 64 + 1024;             // + slack for the 1024-byte alignment of the tiles
  static constexpr int kMax = 148 * kCtas;
  static_assert(kOffQ >= 4 * 8 * D * 4, "the four warps' sums");
};

// Units of one (kv head, row tile) of sequence b, and its row tiles.
__device__ __forceinline__ int2 units_of(const Q8View &p, int b) {
  const int rows = rows_of(p, b).y * p.gq;
  return make_int2((tokens_of(p, b) + kFewUnit - 1) / kFewUnit, rows <= p.few_rows ? (rows + 7) / 8 : 0);
}

__device__ __forceinline__ long long seq_units(const Q8View &p, int b) {
  const int2 u = units_of(p, b);
  return static_cast<long long>(u.x) * u.y * p.Hkv;
}

// The units of all sequences, and the sequence that holds unit begin(cta) of
// them with the units before it (B, 0 for a CTA without work).  A CTA-wide
// scan over the sequences, THREADS at a time: once where they are that few.
struct Found {
  int b;
  long long before, total;
};
template <int THREADS>
__device__ Found find_unit(const Q8View &p, int cta, int ctas) {
  constexpr int W = THREADS / 32;
  __shared__ long long s_w[W];
  __shared__ Found s_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  long long mine = 0;  // units of this thread's first sequence
  long long total = 0;
  for (int b = tid; b < p.B; b += THREADS) {
    const long long u = seq_units(p, b);
    if (b == tid) mine = u;
    total += u;
  }
  // Inclusive sums of the first THREADS sequences, and the total.
  long long v = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xFFFFFFFFu, v, off);
    if (lane >= off) v += o;
  }
  if (p.B > THREADS) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
    if (lane == 0) s_w[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) total += s_w[w];
    __syncthreads();
  }
  if (lane == 31) s_w[warp] = v;
  if (tid == 0) s_found = Found{p.B, 0, 0};
  __syncthreads();
  long long before = v - mine, carry = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_w[w];
    carry += s_w[w];
  }
  if (p.B <= THREADS) total = carry;
  const long long start = Ranges(total, ctas).begin(cta);
  if (before <= start && start < before + mine) s_found = Found{tid, before, 0};
  for (int b0 = THREADS; b0 < p.B && carry <= start; b0 += THREADS) {
    const int b = b0 + tid;
    mine = b < p.B ? seq_units(p, b) : 0;
    v = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xFFFFFFFFu, v, off);
      if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 31) s_w[warp] = v;
    __syncthreads();
    before = carry + v - mine;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += s_w[w];
      carry += s_w[w];
    }
    if (before <= start && start < before + mine) s_found = Found{b, before, 0};
  }
  __syncthreads();
  return Found{s_found.b, s_found.before, total};
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kFewThreads, Few<D, E4M3>::kCtas) k_q8_few(Q8View p, const __grid_constant__ CUtensorMap kmap,
                                                                                 const __grid_constant__ CUtensorMap vmap, uint32_t *err) {
  constexpr int VC = D == 64 ? 1 : D / 128;  // pieces of a V row per lane
  constexpr int VW = D == 64 ? 2 : 4;      // words of a V piece
  constexpr int MT = D / 16;               // 16-dim tiles of O^T
  using F = Few<D, E4M3>;
  extern __shared__ uint8_t few_raw[];
  const uint32_t sbase = (smem_u32(few_raw) + 1023u) & ~1023u;
  uint8_t *few_ring = few_raw + (sbase - smem_u32(few_raw));
  float (*s_o)[8][D] = reinterpret_cast<float (*)[8][D]>(few_ring);
  __shared__ float s_m[4][8], s_l[4][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  pdl_wait();
  pdl_trigger();
  const uint32_t kbar = sbase + F::kOffBar + 16 * warp, vbar = kbar + 8;
  if (lane == 0) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(kbar));
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(vbar));
    mbar_init_fence();
  }
  uint32_t phase = 0;  // of both: they complete once a step
  bool dead = false;
  const Found f = find_unit<kFewThreads>(p, blockIdx.x, gridDim.x);
  const Ranges ranges(f.total, gridDim.x);
  long long cur = ranges.begin(blockIdx.x);
  const long long first = cur, end = ranges.begin(blockIdx.x + 1);
  int b = f.b;
  long long off = cur - f.before;  // within the sequence

  while (cur < end) {
    int2 u = units_of(p, b);
    while (off >= static_cast<long long>(u.x) * u.y * p.Hkv) {  // next sequence with work
      off -= static_cast<long long>(u.x) * u.y * p.Hkv;
      u = units_of(p, ++b);
    }
    const int seg = off <= 0xFFFFFFFFll ? static_cast<uint32_t>(off) / static_cast<uint32_t>(u.x) : static_cast<int>(off / u.x);
    const int u0 = static_cast<int>(off - static_cast<long long>(seg) * u.x);
    const int n = static_cast<int>(min(static_cast<long long>(u.x - u0), end - cur));
    const int h = seg / u.y, rt = seg - h * u.y;
    const int2 qr = rows_of(p, b);
    const int ctx = tokens_of(p, b);
    const int rows = qr.y * p.gq;
    const int lim0 = p.ctx[b] - qr.y;  // last position that row 0 sees

    // ---- this warp's steps of 32 tokens ----
    const int t_end = min(ctx, (u0 + n) * kFewUnit);
    int t = u0 * kFewUnit + 32 * warp;
    const int32_t *trow = p.table + static_cast<size_t>(b) * p.width;
    const uint32_t ring = sbase + warp * F::kWarpBytes;
    const uint32_t qat = sbase + F::kOffQ + 8 * lane;
    // This lane's value bytes of tokens 2t, 2t + 1 (tokens + 8 lie half a box on).
    const uint32_t v_off[2] = {D == 64 ? tile_offset<D>(2 * tq, g >> 1) + 8 * (g & 1) : tile_offset<D>(2 * tq, g),
                               D == 64 ? tile_offset<D>(2 * tq + 1, g >> 1) + 8 * (g & 1) : tile_offset<D>(2 * tq + 1, g)};
    constexpr uint32_t kTile1 = D == 64 ? 1024 : 2048;  // from a step's first tile to its second
    const uint32_t kat[2] = {ring, ring + kTile1}, vat[2] = {ring + 2 * F::kTileBytes, ring + 2 * F::kTileBytes + kTile1};
    // The two tiles of the step to request next: their pages (looked up a step
    // ahead; -1 where there is none) and the scales that come with their codes.
    int pg[2], inpage[2], slot[2] = {-1, -1};
    float ks[2], vs[2];
    const float *ks_h = p.ks + h, *vs_h = p.vs + h;
    auto look_up = [&](int tt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int pos = tt + 16 * e, cc = page_col(p, pos);
        inpage[e] = pos - cc * p.page;
        pg[e] = pos < t_end ? trow[cc] : -1;
      }
    };
    // Pages of whole steps: one box of 32 rows for both tiles, else one of 16 each.
    auto request = [&](const CUtensorMap &map, uint32_t dst, uint32_t bar) {
      const int x = h * D;
      if (p.pair_boxes) {
        mbar_expect_tx_u32(bar, slot[0] >= 0 ? 2 * F::kTileBytes : 0);
        if (slot[0] < 0) return;
#pragma unroll
        for (int c = 0; c < (D + 127) / 128; ++c) tma_box2d(dst + 4096 * c, &map, x + 128 * c, slot[0], bar);
      } else {
        mbar_expect_tx_u32(bar, ((slot[0] >= 0) + (slot[1] >= 0)) * F::kTileBytes);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < (D + 127) / 128; ++c)
            if (slot[e] >= 0) tma_box2d(dst + kTile1 * e + 4096 * c, &map, x + 128 * c, slot[e], bar);
      }
    };
    auto request_k = [&](int tt) {
      if (tt >= t_end) return;
#pragma unroll
      for (int e = 0; e < 2; ++e)  // first slot of the tile, or -1 without a page in the cache
        slot[e] = static_cast<uint32_t>(pg[e]) < static_cast<uint32_t>(p.pages) ? pg[e] * p.page + inpage[e] : -1;
      if (lane == 0 && !dead) request(kmap, kat[0], kbar);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint64_t sc = static_cast<uint64_t>(static_cast<uint32_t>(max(slot[e], 0)) >> p.block_shift) * static_cast<uint32_t>(p.Hkv);
        ks[e] = __ldcg(ks_h + sc);
        vs[e] = __ldcg(vs_h + sc);
      }
    };
    auto request_v = [&](int tt) {
      if (tt < t_end && lane == 0 && !dead) request(vmap, vat[0], vbar);
    };
    auto arrived = [&](uint32_t bar) {  // bounded: a copy that never lands sets the error word
      uint32_t spins = 0;
      while (!dead && !mbar_try_wait_u32(bar, phase))
        if (++spins >= kFewSpin) {
          set_error(err, kErrTimeout);
          dead = true;
        }
      dead = __any_sync(0xFFFFFFFFu, dead);
    };
    look_up(t);
    request_k(t);
    request_v(t);
    look_up(t + kFewUnit);

    // ---- this tile's query rows, their scale and the last position each sees ----
    float c[2];
    int lim[2];
    {
      const int r = rt * 8 + g;
      const bool live = r < rows;
      const int qi = live ? r / p.gq : 0;
      const int head = h * p.gq + (live ? r - qi * p.gq : 0);
      const uint16_t *src = p.q + static_cast<uint64_t>(qr.x + qi) * p.q_stride + static_cast<uint64_t>(head) * D + 4 * tq;
      uint2 raw[D / 32][2];
      uint32_t peak = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          raw[i][e] = live ? *reinterpret_cast<const uint2 *>(src + 32 * i + 16 * e) : make_uint2(0, 0);
          peak = max(peak, max(max(raw[i][e].x & 0x7FFFu, (raw[i][e].x >> 16) & 0x7FFFu),
                               max(raw[i][e].y & 0x7FFFu, (raw[i][e].y >> 16) & 0x7FFFu)));
        }
      peak = max(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, 1));
      peak = max(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, 2));
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        if ((i & 3) == warp) F::Query::put(reinterpret_cast<uint2 *>(few_ring + F::kOffQ), i, raw[i][0], raw[i][1], peak);
      const float up = F::Query::scale_of(peak);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        c[hh] = p.scale * kLog2e * __shfl_sync(0xFFFFFFFFu, up, (2 * tq + hh) * 4);
        const int rr = rt * 8 + 2 * tq + hh;
        lim[hh] = rr < rows ? lim0 + rr / p.gq : 0x7FFFFFFF;  // rows past the end: never written
      }
    }

    const int lim_min = __reduce_min_sync(0xFFFFFFFFu, min(lim[0], lim[1]));

    float o[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float v_top = 0.0f;  // the largest value scale so far

    __syncthreads();  // the query rows are in place
    for (; t < t_end; t += kFewUnit) {
      const bool in[2] = {slot[0] >= 0, slot[1] >= 0};
      float sc[2][4];  // (token g, row 2 tq), (g, 2 tq + 1), (g + 8, 2 tq), (g + 8, 2 tq + 1)
      arrived(kbar);
      F::Query::scores(kat, qat, sc);
      const float k_scale[2] = {ks[0], ks[1]};
      float lv[2], rv[2], fold[2];
      v_top = fmaxf(v_top, fmaxf(in[0] ? vs[0] : 0.0f, in[1] ? vs[1] : 0.0f));
      const float v_least = fmaxf(v_top * kScaleSpan, kScaleLeast);
      const bool folds = (in[0] && vs[0] < v_least) || (in[1] && vs[1] < v_least);  // of the whole warp
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v_scale = fmaxf(vs[e], v_least);
        lv[e] = lg2(v_scale);
        rv[e] = rcp(v_scale);
        fold[e] = vs[e] < v_least ? vs[e] * rv[e] : 1.0f;
      }
      __syncwarp();  // every lane has read its K
      request_k(t + kFewUnit);

      // t_j, the running reference, the weights
      float x[2][4];
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float mul = c[hh] * k_scale[e];
          x[e][hh] = __fmaf_rn(sc[e][hh], mul, lv[e]);
          x[e][2 + hh] = __fmaf_rn(sc[e][2 + hh], mul, lv[e]);
        }
      if (!in[0] || !in[1] || t + 31 > lim_min) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (!in[e] || t + 16 * e + g + 8 * (k >> 1) > lim[k & 1]) x[e][k] = -INFINITY;
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) top[hh] = fmaxf(fmaxf(x[0][hh], x[0][2 + hh]), fmaxf(x[1][hh], x[1][2 + hh]));
      if (__any_sync(0xFFFFFFFFu, top[0] > m[0] + kLazy || top[1] > m[1] + kLazy)) {
        float al[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float cm = top[hh];
#pragma unroll
          for (int s = 4; s <= 16; s <<= 1) cm = fmaxf(cm, __shfl_xor_sync(0xFFFFFFFFu, cm, s));
          cm = fmaxf(cm, m[hh]);
          al[hh] = cm == -INFINITY ? 1.0f : ex2(m[hh] - cm);
          if (cm != -INFINITY) l[hh] = times_ex2(l[hh], m[hh] - cm);
          m[hh] = cm;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          o[j][0] *= al[0];
          o[j][1] *= al[1];
          o[j][2] *= al[0];
          o[j][3] *= al[1];
        }
      }
      const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
      uint32_t hi[2][2], lo[2][2];  // [tile][tokens g | g + 8 transposed]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float p0 = ex2(x[e][0] - ref[0]), p1 = ex2(x[e][1] - ref[1]);
        float p2 = ex2(x[e][2] - ref[0]), p3 = ex2(x[e][3] - ref[1]);
        l[0] = __fmaf_rn(p0 + p2, rv[e], l[0]);
        l[1] = __fmaf_rn(p1 + p3, rv[e], l[1]);
        if (folds) {
          p0 *= fold[e];
          p1 *= fold[e];
          p2 *= fold[e];
          p3 *= fold[e];
        }
        split_bf16x2(p0, p1, hi[e][0], lo[e][0]);
        split_bf16x2(p2, p3, hi[e][1], lo[e][1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          hi[e][k] = movm_t(hi[e][k]);
          lo[e][k] = movm_t(lo[e][k]);
        }
      }

      // O^T += V^T P^T.  Slots past the context (or of a page outside the
      // cache) may hold anything and weigh 0; e4m3 codes can be NaN, so those
      // slots' bytes are zeroed.
      arrived(vbar);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int live = in[e] ? min(16, ctx - t - 16 * e) : 0;
        const bool tail = E4M3 && __any_sync(0xFFFFFFFFu, live < 16);
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          uint32_t v[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (D == 64) {
              const uint2 y = lds64(vat[e] + v_off[k & 1] + (k >> 1) * 512);
              v[k][0] = y.x;
              v[k][1] = y.y;
            } else {
              const uint4 y = lds128(vat[e] + v_off[k & 1] + (k >> 1) * 1024 + i * 4096);
              v[k][0] = y.x;
              v[k][1] = y.y;
              v[k][2] = y.z;
              v[k][3] = y.w;
            }
          }
          if (tail) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int w = 0; w < VW; ++w) v[k][w] = 2 * tq + (k & 1) + 8 * (k >> 1) < live ? v[k][w] : 0u;
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t a[4], b4[4];  // [dim of the word]: tokens (2t, 2t+1), tokens (2t+8, 2t+9)
            widen_pairs<E4M3>(v[0][w], v[1][w], a);
            widen_pairs<E4M3>(v[2][w], v[3][w], b4);
            const uint32_t a0[4] = {a[0], a[1], b4[0], b4[1]}, a1[4] = {a[2], a[3], b4[2], b4[3]};
            mma_bf16(o[2 * VW * i + 2 * w], a0, hi[e][0], hi[e][1]);
            mma_bf16(o[2 * VW * i + 2 * w + 1], a1, hi[e][0], hi[e][1]);
            mma_bf16(o[2 * VW * i + 2 * w], a0, lo[e][0], lo[e][1]);
            mma_bf16(o[2 * VW * i + 2 * w + 1], a1, lo[e][0], lo[e][1]);
          }
        }
      }
      phase ^= 1u;
      __syncwarp();  // every lane has read its V
      request_v(t + kFewUnit);
      look_up(t + 2 * kFewUnit);
    }

    // ---- join the four warps ----
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
      for (int s = 4; s <= 16; s <<= 1) l[hh] += __shfl_xor_sync(0xFFFFFFFFu, l[hh], s);
      if (g == 0) {
        s_m[warp][2 * tq + hh] = m[hh];
        s_l[warp][2 * tq + hh] = l[hh];
      }
    }
    if (threadIdx.x == 0) {
      const bool cut = cur == first && u0 > 0, done = u0 == 0 && n == u.x;
      const long long a = cur - u0;
      if (p.by_seg ? cut || done : cur == first) {
        const int4 c4 = cut ? cut_of(ranges, b, h, rt, a, a, a + u.x - 1, blockIdx.x) : make_int4(-1, 0, 0, 0);
        // by segment: only the first cut in it (or the one CTA that did it all) says so
        if (!p.by_seg) p.cuts[blockIdx.x] = c4;
        else if (!cut || c4.x >= 0) p.cuts[(static_cast<size_t>(b) * p.Hkv + h) * p.few_tiles + rt] = make_int4(c4.x, blockIdx.x - 1, c4.z, c4.w);
      }
    }
    __syncthreads();  // also: every warp is done with its ring
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = 2 * tq + hh;
      const float mm = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
      const float fac = m[hh] == -INFINITY ? 0.0f : ex2(m[hh] - mm);
#pragma unroll
      for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const float *a = o[2 * VW * i + 2 * w], *bb = o[2 * VW * i + 2 * w + 1];
          *reinterpret_cast<float4 *>(&s_o[warp][r][128 * i + 4 * VW * g + 4 * w]) =
              make_float4(a[hh] * fac, a[2 + hh] * fac, bb[hh] * fac, bb[2 + hh] * fac);
        }
    }
    __syncthreads();
    const bool whole = u0 == 0 && n == u.x;
    const int part_slot = 2 * blockIdx.x + (cur == first ? 0 : 1);
    for (int i = threadIdx.x; i < 8 * D / 4; i += kFewThreads) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      const int rr = rt * 8 + r;
      if (rr >= rows) continue;
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w][r]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 v = *reinterpret_cast<const float4 *>(&s_o[w][r][d]);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
        if (s_m[w][r] != -INFINITY) ll += times_ex2(s_l[w][r], s_m[w][r] - mm);
      }
      if (whole) {
        const float inv = ll > 0.0f ? __frcp_rn(ll) : 0.0f;
        const int qi = rr / p.gq, head = h * p.gq + rr - qi * p.gq;
        *reinterpret_cast<uint2 *>(p.out + (static_cast<size_t>(qr.x + qi) * p.Hq + head) * D + d) =
            make_uint2(pack_bf16x2(s.x * inv, s.y * inv), pack_bf16x2(s.z * inv, s.w * inv));
      } else {
        *reinterpret_cast<float4 *>(p.part + (static_cast<size_t>(part_slot) * 8 + r) * D + d) = s;
        if (d == 0) p.part_ml[part_slot * 8 + r] = make_float2(mm, ll);
      }
    }
    fence_proxy_async();  // the next piece's copies land where the sums were
    __syncthreads();      // and s_m, s_l and s_o are rewritten
    cur += n;
    off += n;
  }
  if (dead)  // give what is still in flight as long again before the CTA may end
    for (uint32_t spins = 0; spins < kFewSpin && !(mbar_try_wait_u32(kbar, phase) && mbar_try_wait_u32(vbar, phase)); ++spins) {
    }
  if (first >= end && threadIdx.x == 0 && !p.by_seg) p.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  // rows of sequences without a token
  for (int e = blockIdx.x; e < p.B; e += gridDim.x) {
    const int2 u = units_of(p, e);
    if (u.x != 0 || u.y == 0) continue;
    const int2 qr = rows_of(p, e);
    uint2 *dst = reinterpret_cast<uint2 *>(p.out + static_cast<size_t>(qr.x) * p.Hq * D);
    for (int i = threadIdx.x; i < qr.y * p.Hq * (D / 4); i += kFewThreads) dst[i] = make_uint2(0, 0);
  }
  if (p.cu == nullptr) return;
  // rows of no sequence: before the first one's and past the last one's
  const uint64_t row = static_cast<uint64_t>(p.Hq) * (D / 8);
  const uint64_t ahead = row * static_cast<uint64_t>(min(max(p.cu[0], 0), p.rows));
  const uint64_t after = row * static_cast<uint64_t>(min(max(p.cu[p.B], 0), p.rows)), all = row * static_cast<uint64_t>(p.rows);
  uint4 *dst = reinterpret_cast<uint4 *>(p.out);
  const uint64_t i0 = static_cast<uint64_t>(blockIdx.x) * kFewThreads + threadIdx.x, step = static_cast<uint64_t>(gridDim.x) * kFewThreads;
  for (uint64_t i = i0; i < ahead; i += step) dst[i] = make_uint4(0, 0, 0, 0);
  for (uint64_t i = after + i0; i < all; i += step) dst[i] = make_uint4(0, 0, 0, 0);
}

// Joins the sums of segments that several CTAs worked on, in CTA order.  A CTA
// takes one of the eight rows of a few-row segment, or four of the 128 rows of
// a many-row one (cut tiles keep four dims of four rows together).  It finds
// the cut by the segment where there are fewer of those than CTAs to cut them
// (by_seg), else by the CTA whose range it begins.  A CTA's first piece of work
// is in workspace slot 2c, a later cut one in 2c + 1.
template <int D>
__global__ void __launch_bounds__(256) k_q8_join(Q8View p, int few, int many) {
  constexpr int L = D / 4;
  __shared__ float4 s_o[256];
  __shared__ float s_l[256];
  pdl_wait();
  pdl_trigger();
  const bool is_few = static_cast<int>(blockIdx.x) < p.join_rows * few;
  const int at = is_few ? blockIdx.x / p.join_rows : (blockIdx.x - p.join_rows * few) >> 5;
  const int row0 = is_few ? blockIdx.x % p.join_rows : 4 * ((blockIdx.x - p.join_rows * few) & 31);
  const bool by_seg = is_few ? p.by_seg : p.tby_seg;
  int4 cut;
  int c0, h;
  if (by_seg) {
    cut = (is_few ? p.cuts : p.tcuts)[at];
    h = is_few ? at / p.few_tiles % p.Hkv : at % p.Hkv;
    c0 = cut.y;
    if (is_few) {  // segments without rows or tokens were not written
      const int b = at / (p.few_tiles * p.Hkv), rows = rows_of(p, b).y * p.gq;
      if (tokens_of(p, b) == 0 || rows > p.few_rows || at % p.few_tiles * 8 >= rows) return;
    } else if (at / p.Hkv >= p.seq_tile[p.B] || p.tiles[at / p.Hkv].z == 0) {
      return;
    }
  } else {
    cut = (is_few ? p.cuts : p.tcuts)[at + 1];
    h = cut.y;
    c0 = at;
  }
  // Not cut; or never written, where a kernel gave up a wait (its device error is set).
  // (By segment h is in range; its divisions are still under way, and waiting for them here
  // costs 64 ragged sequences 1.3 us.)
  if (!cut_fits(cut, c0, by_seg ? 0 : h, p.B, p.Hkv, is_few ? p.ctas : p.tctas)) return;
  const int c1 = last_cta(cut);
  const bool late0 = (cut.w >> 30) & 1;
  const int2 qr = rows_of(p, cut.x);
  const int R = is_few ? 8 : 128;
  if (static_cast<long long>(cut.z) * R + row0 >= static_cast<long long>(qr.y) * p.gq) return;
  const int rows = qr.y * p.gq - cut.z * R;
  // sub: which of the rows taken at once; lane: four dims; every `groups`-th CTA
  const int per = is_few ? 1 : 4, groups = 256 / (L * per) > 0 ? 256 / (L * per) : 1;
  const int sub = is_few ? 0 : threadIdx.x & 3;
  const int lane = is_few ? threadIdx.x % L : (threadIdx.x >> 2) % L;
  const int grp = threadIdx.x / (L * per), r = row0 + sub;
  const float2 *ml_all = is_few ? p.part_ml : p.tpart_ml;
  auto slot_of = [&](int c) { return static_cast<size_t>(2 * c + (c == c0 && late0 ? 1 : 0)); };
  float mm = -INFINITY;  // over the CTAs: a lane (or four, one a row) takes every 32nd (8th)
  const int wl = threadIdx.x & 31;
  for (int c = c0 + (is_few ? wl : wl >> 2); c <= c1; c += is_few ? 32 : 8) mm = fmaxf(mm, ml_all[slot_of(c) * R + r].x);
  if (is_few) {
    mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, 1));
    mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, 2));
  }
#pragma unroll
  for (int s = 4; s <= 16; s <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, s));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float ll = 0.0f;
  // CTAs whose sums are asked for at once.  (1: verify of 16 sequences 91 us, prefill chunk 368;
  // 2: 89 and 368; 4: 88 and 373; 8: 91 and 393.)
  constexpr int kAhead = 2;
  for (int c = c0 + grp; c <= c1; c += kAhead * groups) {
    float2 ml[kAhead];
    float4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      ml[k] = make_float2(-INFINITY, 0.0f);
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c + k * groups <= c1) {
        const size_t s = slot_of(c + k * groups);
        ml[k] = ml_all[s * R + r];
        v[k] = is_few ? *reinterpret_cast<const float4 *>(p.part + (s * 8 + r) * D + 4 * lane)
                      : reinterpret_cast<const float4 *>(p.tpart)[(s * L + lane) * 128 + r];
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float half = ml[k].x == -INFINITY ? 0.0f : ex2(0.5f * (ml[k].x - mm)), w = half * half;
      ll += ml[k].y * half * half;  // as times_ex2
      acc.x += v[k].x * w;
      acc.y += v[k].y * w;
      acc.z += v[k].z * w;
      acc.w += v[k].w * w;
    }
  }
  if (groups > 1) {
    s_o[threadIdx.x] = acc;
    s_l[threadIdx.x] = ll;
    __syncthreads();
    if (grp != 0) return;
    for (int g = 1; g < groups; ++g) {
      const float4 v = s_o[threadIdx.x + g * L * per];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
      ll += s_l[threadIdx.x + g * L * per];
    }
  }
  if (r >= rows) return;
  const int rr = cut.z * R + r, qi = rr / p.gq, head = h * p.gq + rr - qi * p.gq;
  const float inv = ll > 0.0f ? __frcp_rn(ll) : 0.0f;
  *reinterpret_cast<uint2 *>(p.out + (static_cast<size_t>(qr.x + qi) * p.Hq + head) * D + 4 * lane) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Tokens of a table row: positions are ints, and the kernels look up to three steps of 128 ahead.
constexpr uint64_t kMostTokens = (1ull << 31) - 1024;

int check(const FnQ8AttentionArgs *a, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (const int rc = check_q8_cache(a->cache, err)) return rc;
  const FnQ8Cache &c = a->cache;
  if (a->batch == 0 || a->batch > 0x7FFFFFFFu || a->max_pages == 0 || a->q_rows > 0x7FFFFFFFu || a->q_heads == 0 ||
      a->q_heads % c.kv_heads || static_cast<uint64_t>(a->max_pages) * c.page_size > kMostTokens ||
      (a->cu_q == nullptr && a->q_rows != a->batch)) {
    err = "attention needs sequences, a table row of at most 2^31 - 1024 tokens, q_heads a multiple of kv_heads and, "
          "without cu_q, one row per sequence";
    return FNMOE_ERR_SHAPE;
  }
  if (static_cast<uint64_t>(a->q_rows) * (a->q_heads / c.kv_heads) > 0x7FFFFF00ull) {
    err = "too many query rows";
    return FNMOE_ERR_SHAPE;
  }
  if (a->q_heads / c.kv_heads > 32) { err = "at most 32 query heads per kv head"; return FNMOE_ERR_UNSUPPORTED; }
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) { err = "scale must be finite and positive"; return FNMOE_ERR_VALUE; }
  if (a->q_rows == 0) return FNMOE_OK;
  if (!a->q || !a->block_table || !a->context_lens || !a->out) {
    err = "q, block_table, context_lens and out are required";
    return FNMOE_ERR_NULL;
  }
  if (a->q_stride < static_cast<uint64_t>(a->q_heads) * c.head_dim) {
    err = "q_stride must cover a row of q_heads * head_dim values";
    return FNMOE_ERR_SHAPE;
  }
  if (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15u) || a->q_stride % 8) {
    err = "q and out must be 16-byte aligned and q_stride a multiple of 8 values";
    return FNMOE_ERR_VALUE;
  }
  if ((reinterpret_cast<uintptr_t>(a->block_table) | reinterpret_cast<uintptr_t>(a->context_lens) |
       reinterpret_cast<uintptr_t>(a->cu_q)) & 3u) {
    err = "block_table, context_lens and cu_q must be 4-byte aligned";
    return FNMOE_ERR_VALUE;
  }
  return FNMOE_OK;
}

uint64_t align256(uint64_t n) { return (n + 255) & ~static_cast<uint64_t>(255); }

// Workspace: prefix sums and tiles, then the cut segments' sums.
struct Carve {
  uint64_t cuts, ml, part, seq_tile, tiles, tprefix, tcuts, tml, tpart, bytes;
};
Carve carve(const FnQ8AttentionArgs *a, const Q8View &p, bool few, bool many) {
  const uint64_t d = a->cache.head_dim;
  const uint64_t slots = few ? 2ull * few_ctas(static_cast<int>(d)) : 0;
  const uint64_t tiles = many ? many_tiles(p) : 0, tslots = many ? 2ull * many_ctas(static_cast<int>(d)) : 0;
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t here = at;
    at += align256(n);
    return here;
  };
  Carve c{};
  c.cuts = take(slots / 2 * sizeof(int4));
  c.ml = take(slots * 8 * sizeof(float2));
  c.part = take(slots * 8 * d * sizeof(float));
  c.seq_tile = take(4 * (static_cast<uint64_t>(a->batch) + 1));
  c.tiles = take(sizeof(int4) * tiles);
  c.tprefix = take(8 * (tiles + 1));
  c.tcuts = take(tslots / 2 * sizeof(int4));
  c.tml = take(tslots * 128 * sizeof(float2));
  c.tpart = take(tslots * 128 * d * sizeof(float));
  c.bytes = at + 256;  // the start is rounded up to 256 bytes
  return c;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no -lcuda).
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn q8_encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// Codes as a byte matrix [slots][Hkv * D]: boxes of 16 (pair: 32) slots x 128 (or 64) bytes.
bool make_codes_map(CUtensorMap *map, const void *base, uint64_t slots, uint64_t cols, int D, bool pair) {
  EncodeTiledFn fn = q8_encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {cols, slots};
  const cuuint64_t strides[1] = {cols};
  const cuuint32_t box[2] = {D == 64 ? 64u : 128u, pair ? 32u : 16u};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
            // no more than the head's own bytes: its neighbours' are read by others at other times
            D == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B : D == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool E4M3>
cudaError_t launch_few(const Q8View &p, cudaStream_t s) {
  using F = Few<D, E4M3>;
  CUtensorMap km, vm;
  const uint64_t slots = static_cast<uint64_t>(p.pages) * p.page, cols = static_cast<uint64_t>(p.Hkv) * D;
  if (!make_codes_map(&km, p.kc, slots, cols, D, p.pair_boxes) || !make_codes_map(&vm, p.vc, slots, cols, D, p.pair_boxes)) return cudaErrorInvalidValue;
  static SmemLimit limit;
  const cudaError_t e = limit.set(reinterpret_cast<const void *>(k_q8_few<D, E4M3>), F::kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_q8_few<D, E4M3>, dim3(F::kMax), dim3(kFewThreads), F::kSmem, s, p, km, vm, device_error_word());
}

template <int D>
cudaError_t launch_joins(const Q8View &p, int few, int many, cudaStream_t s) {
  return launch_pdl(k_q8_join<D>, dim3(p.join_rows * few + 32 * many), dim3(256), 0, s, p, few, many);
}

template <int D>
cudaError_t launch_few_d(const Q8View &p, bool e4m3, cudaStream_t s) {
  return e4m3 ? launch_few<D, true>(p, s) : launch_few<D, false>(p, s);
}

Q8View view_of(const FnQ8AttentionArgs *a) {
  const FnQ8Cache &c = a->cache;
  Q8View p{};
  p.q = static_cast<const uint16_t *>(a->q);
  p.kc = static_cast<const uint8_t *>(c.k_codes);
  p.vc = static_cast<const uint8_t *>(c.v_codes);
  p.ks = c.k_scale;
  p.vs = c.v_scale;
  p.table = a->block_table;
  p.ctx = a->context_lens;
  p.cu = a->cu_q;
  p.out = static_cast<uint16_t *>(a->out);
  p.q_stride = a->q_stride;
  p.B = static_cast<int>(a->batch);
  p.rows = static_cast<int>(a->q_rows);
  p.Hq = static_cast<int>(a->q_heads);
  p.Hkv = static_cast<int>(c.kv_heads);
  p.gq = p.Hq / p.Hkv;
  p.page = static_cast<int>(c.page_size);
  p.block_shift = 31 - __builtin_clz(c.block);
  p.width = static_cast<int>(a->max_pages);
  p.pages = static_cast<int>(c.num_pages);
  p.page_magic = static_cast<uint32_t>(((1ull << 32) + c.page_size - 1) / c.page_size);
  p.scale = a->scale;
  p.few_rows = kFewRows;
  p.pair_boxes = c.page_size % 32 == 0;
  return p;
}

// Which kernels a call can need: a sequence's rows are not known on the host,
// but without cu_q each has one, and no sequence has more than all of them.
bool wants_few(const Q8View &p) { return p.cu != nullptr || p.gq <= p.few_rows; }
bool wants_many(const Q8View &p) {
  return p.cu != nullptr ? static_cast<uint64_t>(p.rows) * p.gq > static_cast<uint64_t>(p.few_rows) : p.gq > p.few_rows;
}

}  // namespace

int few_ctas(int head_dim) {
  return head_dim == 256 ? Few<256, false>::kMax : head_dim == 128 ? Few<128, false>::kMax : Few<64, false>::kMax;
}

int paged_attention_q8_workspace_size(const FnQ8AttentionArgs *a, uint64_t *bytes, std::string &err) {
  if (bytes == nullptr) { err = "bytes is NULL"; return FNMOE_ERR_NULL; }
  if (const int rc = check(a, err)) return rc;
  const Q8View p = view_of(a);
  *bytes = carve(a, p, wants_few(p), wants_many(p)).bytes;
  return FNMOE_OK;
}

int paged_attention_q8(const FnQ8AttentionArgs *a, cudaStream_t s, std::string &err) {
  if (const int rc = check(a, err)) return rc;
  if (a->q_rows == 0) return FNMOE_OK;
  Q8View p = view_of(a);
  const bool few = wants_few(p), many = wants_many(p);
  const Carve w = carve(a, p, few, many);
  if (a->workspace == nullptr || a->workspace_bytes < w.bytes) {
    err = "workspace needs " + std::to_string(w.bytes) + " bytes";
    return FNMOE_ERR_WORKSPACE;
  }
  uint8_t *ws = reinterpret_cast<uint8_t *>(align256(reinterpret_cast<uintptr_t>(a->workspace)));
  p.cuts = reinterpret_cast<int4 *>(ws + w.cuts);
  p.tcuts = reinterpret_cast<int4 *>(ws + w.tcuts);
  p.part_ml = reinterpret_cast<float2 *>(ws + w.ml);
  p.part = reinterpret_cast<float *>(ws + w.part);
  p.max_tiles = many ? static_cast<int>(many_tiles(p)) : 0;
  p.seq_tile = reinterpret_cast<int *>(ws + w.seq_tile);
  p.tiles = reinterpret_cast<int4 *>(ws + w.tiles);
  p.tprefix = reinterpret_cast<long long *>(ws + w.tprefix);
  p.tpart_ml = reinterpret_cast<float2 *>(ws + w.tml);
  p.tpart = reinterpret_cast<float *>(ws + w.tpart);
  const int d = static_cast<int>(a->cache.head_dim);
  // Segments there can be: the join looks at those where they are fewer than the cuts.
  p.few_tiles = (std::min(p.few_rows, p.cu ? p.few_rows : p.gq) + 7) / 8;
  p.join_rows = p.cu ? 8 : std::min(p.gq, 8);
  const uint64_t few_segs = static_cast<uint64_t>(p.B) * p.Hkv * p.few_tiles;
  const uint64_t many_segs = many ? many_tiles(p) * p.Hkv : 0;
  p.ctas = few_ctas(d);
  p.tctas = many_ctas(d);
  p.by_seg = few_segs < static_cast<uint64_t>(few_ctas(d) - 1);
  p.tby_seg = many_segs < static_cast<uint64_t>(many_ctas(d) - 1);
  const bool e4m3 = a->cache.code_type == FNMOE_Q8_E4M3;
  cudaError_t e = cudaSuccess;
  if (many) e = launch_many(p, d, e4m3, s);
  if (e == cudaSuccess && few)
    e = d == 64    ? launch_few_d<64>(p, e4m3, s)
        : d == 128 ? launch_few_d<128>(p, e4m3, s)
                   : launch_few_d<256>(p, e4m3, s);
  const int few_cuts = !few ? 0 : p.by_seg ? static_cast<int>(few_segs) : few_ctas(d) - 1;
  const int many_cuts = !many ? 0 : p.tby_seg ? static_cast<int>(many_segs) : many_ctas(d) - 1;
  if (e == cudaSuccess)
    e = d == 64    ? launch_joins<64>(p, few_cuts, many_cuts, s)
        : d == 128 ? launch_joins<128>(p, few_cuts, many_cuts, s)
                   : launch_joins<256>(p, few_cuts, many_cuts, s);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    err = std::string("paged attention q8: ") + cudaGetErrorString(e);
    return FNMOE_ERR_LAUNCH;
  }
  return FNMOE_OK;
}

}  // namespace fnmoe
