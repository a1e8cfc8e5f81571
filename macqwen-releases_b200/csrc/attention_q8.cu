// attention_q8.cu -- causal attention over the paged 8-bit KV cache (sm_100a):
// the entry points and the kernels for sequences with few query rows (decode).
// The arithmetic: attention_q8.cuh; many rows: attention_q8_many.cu.
#include <cuda_runtime.h>
#include <stdint.h>

#include <cmath>
#include <string>

#include "attention_q8.cuh"
#include "moe_kernels.cuh"
#include "paged_q8.cuh"

namespace fnmoe {

namespace {

// ---- few rows per sequence --------------------------------------------------
//
// Bound by HBM (one byte a value, 2 * D * Hkv bytes a token).  Work is cut
// into units of 64 tokens of one (sequence, kv head, tile of 8 rows); the
// units of all sequences, laid end to end, are dealt to the CTAs in equal
// contiguous ranges, so ragged contexts load every SM alike.  A CTA's range
// covers whole segments, which it finishes, and at most two cut ones (its
// first and last), whose sums go to the workspace for k_q8_few_join.
//
// A warp takes 16 tokens at a time.  Each lane copies exactly the codes that it
// will feed to its MMA fragments (cp.async into a ring of its own, kStages
// steps deep), so the copies need no swizzle and no barrier, and the ring,
// not the register file, holds the bytes in flight that HBM's latency asks
// for:
//   S^T = K Q^T   (m16n8k16, M = 16 tokens, N = 8 rows): the order of the
//     contraction is free, so lane (g, t) takes 16 consecutive dims of tokens
//     g and g + 8, one 16-byte load for four k-steps;
//   O^T += V^T P^T (M = 16 dims, N = 8 rows, K = 16 tokens): lane (g, t)
//     loads 16 consecutive dims of tokens 2t, 2t+1, 2t+8, 2t+9 and pairs the
//     tokens' bytes with prmt.
// 16 tokens lie in one page and one scale block.

constexpr int kFewThreads = 128;  // 4 warps x 16 tokens = a unit
constexpr int kFewRows = 16;

template <int D>
struct Few {
  static constexpr int kCtas = D == 256 ? 3 : D == 128 ? 4 : 6;  // per SM
  static constexpr int kStages = D == 256 ? 2 : D == 128 ? 3 : 4;
  static constexpr int kHalf = 16 * D;                          // bytes of a step's K (or V) codes
  static constexpr int kWarpBytes = kStages * 2 * kHalf;        // 12 warps or more: 192 KB an SM
  static constexpr int kSmem = 4 * kWarpBytes;                  // the warps' sums are joined in the same space
  static constexpr int kMax = 148 * kCtas;
  static_assert(kSmem >= 4 * 8 * D * 4, "the four warps' sums");
};

// Units of one (kv head, row tile) of sequence b, and its row tiles.
__device__ __forceinline__ int2 units_of(const Q8View &p, int b) {
  const int rows = rows_of(p, b).y * p.gq;
  return make_int2((tokens_of(p, b) + kUnit - 1) / kUnit, rows <= p.few_rows ? (rows + 7) / 8 : 0);
}

// The sequence that holds this CTA's first unit, the units before that
// sequence and the total.  Every thread gets the result.
struct Found {
  int b;
  long long before, total;
};
__device__ __forceinline__ long long seq_units(const Q8View &p, int b) {
  const int2 u = units_of(p, b);
  return static_cast<long long>(u.x) * u.y * p.Hkv;
}

template <int THREADS>
__device__ Found find_unit(const Q8View &p, int cta, int ctas, long long &start, long long &end) {
  __shared__ long long s_w[THREADS / 32];
  __shared__ long long s_before;
  __shared__ int s_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  long long total = 0;
  for (int b = tid; b < p.B; b += THREADS) total += seq_units(p, b);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
  if (lane == 0) s_w[warp] = total;
  if (tid == 0) {
    s_b = p.B;
    s_before = 0;
  }
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) total += s_w[w];
  const int used = ranges_of(total, ctas);
  start = range_start(total, used, cta);
  end = range_start(total, used, cta + 1);
  long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = b0 + tid;
    const long long u = b < p.B ? seq_units(p, b) : 0;
    long long v = u;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xFFFFFFFFu, v, off);
      if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 31) s_w[warp] = v;
    __syncthreads();
    long long before = carry;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += s_w[w];
      carry += s_w[w];
    }
    before += v - u;
    if (b < p.B && before <= start && start < before + u) {
      s_b = b;
      s_before = before;
    }
    if (carry > start) break;
  }
  __syncthreads();
  return Found{s_b, s_before, total};
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kFewThreads, Few<D>::kCtas) k_q8_few(Q8View p) {
  constexpr int KC = D / 64;               // 16-byte pieces of a K row per lane
  constexpr int VC = D == 64 ? 1 : D / 128;  // pieces of a V row per lane
  constexpr int VW = D == 64 ? 2 : 4;      // words of a V piece
  constexpr int MT = D / 16;               // 16-dim tiles of O^T
  using F = Few<D>;
  extern __shared__ __align__(16) uint8_t few_ring[];
  float (*s_o)[8][D] = reinterpret_cast<float (*)[8][D]>(few_ring);
  __shared__ float s_m[4][8], s_l[4][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  pdl_wait();  // launched after the many-row kernel, whose workspace the join reads
  pdl_trigger();
  long long cur, end;
  const Found f = find_unit<kFewThreads>(p, blockIdx.x, gridDim.x, cur, end);
  const long long first = cur;
  int b = f.b;
  long long off = cur - f.before;  // within the sequence

  while (cur < end) {
    int2 u = units_of(p, b);
    while (off >= static_cast<long long>(u.x) * u.y * p.Hkv) {  // next sequence with work
      off -= static_cast<long long>(u.x) * u.y * p.Hkv;
      u = units_of(p, ++b);
    }
    const int seg = static_cast<int>(off / u.x);
    const int u0 = static_cast<int>(off - static_cast<long long>(seg) * u.x);
    const int n = static_cast<int>(min(static_cast<long long>(u.x - u0), end - cur));
    const int h = seg / u.y, rt = seg - h * u.y;
    const int2 qr = rows_of(p, b);
    const int ctx = tokens_of(p, b);
    const int rows = qr.y * p.gq;
    const int lim0 = p.ctx[b] - qr.y;  // last position that row 0 sees

    // ---- this tile's query rows as the B operand, and the last position each sees ----
    uint32_t qf[MT][2];
    int lim[2];
    {
      const int r = rt * 8 + g;
      const bool live = r < rows;
      const int qi = live ? r / p.gq : 0;
      const int head = h * p.gq + (live ? r - qi * p.gq : 0);
      const uint16_t *src = p.q + static_cast<uint64_t>(qr.x + qi) * p.q_stride + static_cast<uint64_t>(head) * D + 16 * tq;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        uint4 w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w[e] = live ? *reinterpret_cast<const uint4 *>(src + 64 * i + 8 * e) : make_uint4(0, 0, 0, 0);
        qf[4 * i][0] = w[0].x;
        qf[4 * i][1] = w[0].y;
        qf[4 * i + 1][0] = w[0].z;
        qf[4 * i + 1][1] = w[0].w;
        qf[4 * i + 2][0] = w[1].x;
        qf[4 * i + 2][1] = w[1].y;
        qf[4 * i + 3][0] = w[1].z;
        qf[4 * i + 3][1] = w[1].w;
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int rr = rt * 8 + 2 * tq + hh;
        lim[hh] = rr < rows ? lim0 + rr / p.gq : -1;
      }
    }

    float o[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    // ---- this warp's 16-token steps ----
    const int t_end = min(ctx, (u0 + n) * kUnit);
    int t = u0 * kUnit + 16 * warp;
    const int32_t *trow = p.table + static_cast<size_t>(b) * p.width;
    const int bpp = p.page >> p.block_shift;
    // Where step t's tokens are: the table column, then (a step later) the page.
    int col = page_col(p, t), at = t - col * p.page;
    int ft = t;          // the next step to request, its column and place in the page
    int fpg = ft < t_end ? trow[col] : -1;  // its page
    const uint32_t row_bytes = static_cast<uint32_t>(p.Hkv) * D;
    const uint32_t ring = smem_u32(few_ring) + warp * F::kWarpBytes;
    const uint8_t *kbase = p.kc + static_cast<size_t>(h) * D + static_cast<size_t>(g) * row_bytes + 16 * tq;
    const uint8_t *vbase = p.vc + static_cast<size_t>(h) * D + static_cast<size_t>(2 * tq) * row_bytes + (D == 64 ? 8 : 16) * g;
    float ks[F::kStages], vs[F::kStages];  // scales of the requested steps, oldest first
    bool ok[F::kStages];                   // and whether their page is in the cache
    auto row_of = [&]() {  // a page outside the cache: page 0 is read and its tokens masked
      const bool in = static_cast<uint32_t>(fpg) < static_cast<uint32_t>(p.pages);
      return static_cast<uint64_t>((in ? static_cast<uint32_t>(fpg) : 0u) * static_cast<uint32_t>(p.page) + static_cast<uint32_t>(at)) * row_bytes;
    };
    auto request_k = [&](uint32_t slot, int e) {
      if (ft < t_end) {
        const uint8_t *src = kbase + row_of();
        const uint32_t dst = ring + slot * (2 * F::kHalf) + 16 * lane;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          cp_async16_u32(dst + (2 * i) * 512, src + 64 * i);
          cp_async16_u32(dst + (2 * i + 1) * 512, src + 64 * i + 8ull * row_bytes);
        }
        ok[e] = static_cast<uint32_t>(fpg) < static_cast<uint32_t>(p.pages);
        const size_t sc = (static_cast<size_t>(ok[e] ? fpg : 0) * bpp + (at >> p.block_shift)) * p.Hkv + h;
        ks[e] = __ldg(p.ks + sc);
        vs[e] = __ldg(p.vs + sc);
      }
      cp_async_commit();
    };
    auto request_v = [&](uint32_t slot) {  // and on to the next step
      if (ft < t_end) {
        const uint8_t *src = vbase + row_of();
        const uint32_t dst = ring + slot * (2 * F::kHalf) + F::kHalf + (D == 64 ? 8 : 16) * lane;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint8_t *r = src + static_cast<uint64_t>((k & 1) + 8 * (k >> 1)) * row_bytes;
          if (D == 64) {
            cp_async8_u32(dst + k * 256, r);
          } else {
#pragma unroll
            for (int i = 0; i < VC; ++i) cp_async16_u32(dst + (k * VC + i) * 512, r + 128 * i);
          }
        }
        ft += kUnit;
        at += kUnit;
        while (at >= p.page) {
          at -= p.page;
          ++col;
        }
        fpg = ft < t_end ? trow[col] : -1;
      }
      cp_async_commit();
    };
#pragma unroll
    for (int e = 0; e < F::kStages; ++e) {
      request_k(e, e);
      request_v(e);
    }
    uint32_t slot = 0;
    for (; t < t_end; t += kUnit) {
      const uint32_t kst = ring + slot * (2 * F::kHalf), vst = kst + F::kHalf;
      // Groups in flight behind this step's K: its V and the steps after it.
      cp_async_wait<2 * F::kStages - 1>();
      // S^T = K Q^T, two chains
      float sa[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sb[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint4 k0 = lds128(kst + 16 * lane + (2 * i) * 512), k1 = lds128(kst + 16 * lane + (2 * i + 1) * 512);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w};
        const uint32_t w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x0 = w0[j], x1 = w1[j];
          const uint32_t a[4] = {widen2<E4M3, 0>(x0), widen2<E4M3, 0>(x1), widen2<E4M3, 1>(x0), widen2<E4M3, 1>(x1)};
          mma_bf16(j & 1 ? sb : sa, a, qf[4 * i + j][0], qf[4 * i + j][1]);
        }
      }
      const float k_scale = ks[0], v_raw = vs[0];
      const bool in = ok[0];
#pragma unroll
      for (int e = 0; e + 1 < F::kStages; ++e) {
        ks[e] = ks[e + 1];
        vs[e] = vs[e + 1];
        ok[e] = ok[e + 1];
      }
      request_k(slot, F::kStages - 1);

      // t_j, the running reference, the weights
      const float v_scale = fmaxf(v_raw, 0x1p-110f);
      const float lv = __log2f(v_scale), rv = __frcp_rn(v_scale);
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = t + g + 8 * (e >> 1), hh = e & 1;
        const float s = __fadd_rn(sa[e], sb[e]);
        x[e] = in && tok <= lim[hh] ? __fmaf_rn(s, p.scale * kLog2e * k_scale, lv) : -INFINITY;
      }
      if (__any_sync(0xFFFFFFFFu, fmaxf(x[0], x[2]) > m[0] + kLazy || fmaxf(x[1], x[3]) > m[1] + kLazy)) {
        float al[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float cm = fmaxf(x[hh], x[hh + 2]);
#pragma unroll
          for (int s = 4; s <= 16; s <<= 1) cm = fmaxf(cm, __shfl_xor_sync(0xFFFFFFFFu, cm, s));
          cm = fmaxf(cm, m[hh]);
          al[hh] = cm == -INFINITY ? 1.0f : ex2(m[hh] - cm);
          m[hh] = cm;
          l[hh] *= al[hh];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          o[j][0] *= al[0];
          o[j][1] *= al[1];
          o[j][2] *= al[0];
          o[j][3] *= al[1];
        }
      }
      const float r0 = m[0] == -INFINITY ? 0.0f : m[0], r1 = m[1] == -INFINITY ? 0.0f : m[1];
      const float p0 = ex2(x[0] - r0), p1 = ex2(x[1] - r1), p2 = ex2(x[2] - r0), p3 = ex2(x[3] - r1);
      l[0] = __fmaf_rn(p0 + p2, rv, l[0]);
      l[1] = __fmaf_rn(p1 + p3, rv, l[1]);
      uint32_t hi0, lo0, hi1, lo1;
      split_bf16x2(p0, p1, hi0, lo0);
      split_bf16x2(p2, p3, hi1, lo1);
      hi0 = movm_t(hi0);
      hi1 = movm_t(hi1);
      lo0 = movm_t(lo0);
      lo1 = movm_t(lo1);

      // Slots past the context (or of a page outside the cache) may hold
      // anything, NaN codes too: their value bytes are zeroed.
      const int live = in ? min(16, ctx - t) : 0;
      uint32_t keep[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = 2 * tq + (k & 1) + 8 * (k >> 1) < live ? 0xFFFFFFFFu : 0u;
      // O^T += V^T P^T
      cp_async_wait<2 * F::kStages - 1>();
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        uint32_t v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (D == 64) {
            const uint2 y = lds64(vst + 8 * lane + k * 256);
            v[k][0] = y.x;
            v[k][1] = y.y;
          } else {
            const uint4 y = lds128(vst + 16 * lane + (k * VC + i) * 512);
            v[k][0] = y.x;
            v[k][1] = y.y;
            v[k][2] = y.z;
            v[k][3] = y.w;
          }
        }
        if (live < 16) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int w = 0; w < VW; ++w) v[k][w] &= keep[k];
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t la = prmt(v[0][w], v[1][w], 0x5140u), ha = prmt(v[0][w], v[1][w], 0x7362u);
          const uint32_t lb = prmt(v[2][w], v[3][w], 0x5140u), hb = prmt(v[2][w], v[3][w], 0x7362u);
          const uint32_t a0[4] = {widen2<E4M3, 0>(la), widen2<E4M3, 1>(la), widen2<E4M3, 0>(lb), widen2<E4M3, 1>(lb)};
          const uint32_t a1[4] = {widen2<E4M3, 0>(ha), widen2<E4M3, 1>(ha), widen2<E4M3, 0>(hb), widen2<E4M3, 1>(hb)};
          mma_bf16(o[2 * VW * i + 2 * w], a0, hi0, hi1);
          mma_bf16(o[2 * VW * i + 2 * w + 1], a1, hi0, hi1);
          mma_bf16(o[2 * VW * i + 2 * w], a0, lo0, lo1);
          mma_bf16(o[2 * VW * i + 2 * w + 1], a1, lo0, lo1);
        }
      }
      request_v(slot);
      slot = slot + 1 == F::kStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();

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
    if (cur == first && threadIdx.x == 0) {
      const long long a = cur - u0;
      p.cuts[blockIdx.x] = u0 == 0 ? make_int4(-1, 0, 0, 0) : cut_of(b, h, rt, a, a, a + u.x - 1, f.total, ranges_of(f.total, gridDim.x), blockIdx.x);
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
        if (s_m[w][r] != -INFINITY) ll += s_l[w][r] * ex2(s_m[w][r] - mm);
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
    __syncthreads();  // s_m, s_l and s_o are rewritten by the next piece
    cur += n;
    off += n;
  }
  if (first >= end && threadIdx.x == 0) p.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  // rows of sequences without a token
  for (int e = blockIdx.x; e < p.B; e += gridDim.x) {
    const int2 u = units_of(p, e);
    if (u.x != 0 || u.y == 0) continue;
    const int2 qr = rows_of(p, e);
    uint2 *dst = reinterpret_cast<uint2 *>(p.out + static_cast<size_t>(qr.x) * p.Hq * D);
    for (int i = threadIdx.x; i < qr.y * p.Hq * (D / 4); i += kFewThreads) dst[i] = make_uint2(0, 0);
  }
}

// Joins the sums of segments that several CTAs worked on, in CTA order.  A CTA
// takes two of the eight rows of a few-row cut, or 16 of the 128 rows of a
// many-row cut (four at a time: cut tiles keep four dims of a row together).
// A CTA's first piece of work is in workspace slot 2c, a later cut one in
// 2c + 1.
template <int D>
__global__ void __launch_bounds__(256) k_q8_join(Q8View p, int few_cuts, int many_cuts) {
  constexpr int L = D / 4, G = 256 / L;
  __shared__ float4 s_o[256];
  __shared__ float s_l[256];
  pdl_wait();
  const bool few = static_cast<int>(blockIdx.x) < 4 * few_cuts;
  const int at = few ? blockIdx.x : blockIdx.x - 4 * few_cuts;
  const int c1_cta = few ? at >> 2 : at >> 3;  // the cut is where CTA c1_cta + 1's range begins
  const int4 cut = few ? p.cuts[c1_cta + 1] : p.tcuts[c1_cta + 1];
  if (cut.x < 0) return;
  const int c0 = c1_cta, c1 = cut.w & 0x3FFFFFFF;
  const bool late0 = (cut.w >> 30) & 1;
  const int2 qr = rows_of(p, cut.x);
  const int R = few ? 8 : 128, rows = qr.y * p.gq - cut.z * R;
  const float2 *ml_all = few ? p.part_ml : p.tpart_ml;
  auto slot_of = [&](int c) { return static_cast<size_t>(2 * c + (c == c0 && late0 ? 1 : 0)); };
  // lane: four dims; sub: which row of those taken at once; grp: every G-th CTA
  const int per = few ? 1 : 4, groups = G / per > 0 ? G / per : 1;
  const int sub = few ? 0 : threadIdx.x & 3;
  const int lane = few ? threadIdx.x % L : (threadIdx.x >> 2) % L;
  const int grp = few ? threadIdx.x / L : threadIdx.x / (4 * L);
  const int row_first = few ? 2 * (at & 3) : 16 * (at & 7), row_count = few ? 2 : 16;
  for (int r0 = row_first; r0 < row_first + row_count && r0 < rows; r0 += per) {
    const int r = r0 + sub;
    float mm = -INFINITY;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) mm = fmaxf(mm, ml_all[slot_of(c) * R + r].x);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f;
#pragma unroll 4
    for (int c = c0 + grp; c <= c1; c += groups) {
      const size_t s = slot_of(c);
      const float2 ml = ml_all[s * R + r];
      const float4 v = few ? *reinterpret_cast<const float4 *>(p.part + (s * 8 + r) * D + 4 * lane)
                           : reinterpret_cast<const float4 *>(p.tpart)[(s * L + lane) * 128 + r];
      const float w = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mm);
      ll += ml.y * w;
      acc.x += v.x * w;
      acc.y += v.y * w;
      acc.z += v.z * w;
      acc.w += v.w * w;
    }
    if (groups > 1) {
      const int stride = L * per;
      __syncthreads();
      s_o[threadIdx.x] = acc;
      s_l[threadIdx.x] = ll;
      __syncthreads();
      if (grp == 0)
        for (int g = 1; g < groups; ++g) {
          const float4 v = s_o[threadIdx.x + g * stride];
          acc.x += v.x;
          acc.y += v.y;
          acc.z += v.z;
          acc.w += v.w;
          ll += s_l[threadIdx.x + g * stride];
        }
    }
    if (grp == 0 && r < rows) {
      const int rr = cut.z * R + r, qi = rr / p.gq, head = cut.y * p.gq + rr - qi * p.gq;
      const float inv = ll > 0.0f ? __frcp_rn(ll) : 0.0f;
      *reinterpret_cast<uint2 *>(p.out + (static_cast<size_t>(qr.x + qi) * p.Hq + head) * D + 4 * lane) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    }
  }
}

int check(const FnQ8AttentionArgs *a, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (const int rc = check_q8_cache(a->cache, err)) return rc;
  const FnQ8Cache &c = a->cache;
  if (a->batch == 0 || a->batch > 0x7FFFFFFFu || a->max_pages == 0 || a->q_rows > 0x7FFFFFFFu || a->q_heads == 0 ||
      a->q_heads % c.kv_heads || static_cast<uint64_t>(a->max_pages) * c.page_size > 0x7FFFFFFFull ||
      (a->cu_q == nullptr && a->q_rows != a->batch)) {
    err = "attention needs sequences, a table row below 2^31 tokens, q_heads a multiple of kv_heads and, "
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

template <int D, bool E4M3>
cudaError_t launch_few(const Q8View &p, bool pdl, cudaStream_t s) {
  using F = Few<D>;
  // Set for every call: the attribute belongs to the current device.
  const cudaError_t e = cudaFuncSetAttribute(k_q8_few<D, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
  if (e != cudaSuccess) return e;
  if (pdl) return launch_pdl(k_q8_few<D, E4M3>, dim3(F::kMax), dim3(kFewThreads), F::kSmem, s, p);
  k_q8_few<D, E4M3><<<F::kMax, kFewThreads, F::kSmem, s>>>(p);
  return cudaSuccess;
}

template <int D>
cudaError_t launch_joins(const Q8View &p, int few_cuts, int many_cuts, cudaStream_t s) {
  return launch_pdl(k_q8_join<D>, dim3(4 * few_cuts + 8 * many_cuts), dim3(256), 0, s, p, few_cuts, many_cuts);
}

template <int D>
cudaError_t launch_few_d(const Q8View &p, bool e4m3, bool pdl, cudaStream_t s) {
  return e4m3 ? launch_few<D, true>(p, pdl, s) : launch_few<D, false>(p, pdl, s);
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
  return head_dim == 256 ? Few<256>::kMax : head_dim == 128 ? Few<128>::kMax : Few<64>::kMax;
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
  const bool e4m3 = a->cache.code_type == FNMOE_Q8_E4M3;
  cudaError_t e = cudaSuccess;
  if (many) e = launch_many(p, d, e4m3, s);
  if (e == cudaSuccess && few)
    e = d == 64    ? launch_few_d<64>(p, e4m3, many, s)
        : d == 128 ? launch_few_d<128>(p, e4m3, many, s)
                   : launch_few_d<256>(p, e4m3, many, s);
  const int few_cuts = few ? few_ctas(d) - 1 : 0, many_cuts = many ? many_ctas(d) - 1 : 0;
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
