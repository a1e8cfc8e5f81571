// norm.cu -- rows of hidden states: the residual's addition, the
// root-mean-square norm and the conversion to 8 bits with a scale a row, in
// one pass over the row; and codes back to values.
//
//   s = x + residual
//   y = s / sqrt(mean(s^2) + eps) * w          (w or 1 + w; left out when only quantising)
//   scale = max(max |y|, 2^-100) / top, code = round(y / scale)   (top 127 or 448)
//
// A row is read once and stays in registers.  One reduction finds both sum(s^2)
// and max |s w|: the norm's factor is the same for the whole row, so
// max |y| = max |s w| / rms and the codes need no second reduction.  Sums and y
// are float32; y and the carried residual are rounded once, from float32 (the
// norm sees the unrounded sum, so rounding the carried residual costs it
// nothing).
//
// Bound by issue slots and HBM: CTAs stay on their SM and ask for rows ahead, and
// nothing is chosen a value at a time.  5000 x 2048 bfloat16 with a residual: 17 to 19
// us, 4.3 to 4.8 TB/s of 6.46 (41 instructions a value with codes, 55 in the first
// form); one row of 2048: 2.0 us, of which a launch is most.  Rows off boundaries that
// are not contiguous (kOdd): 69 us padded to 2051, one value a load, and values of
// two chunks that do not fit the registers.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "dense.cuh"
#include "moe_kernels.cuh"

namespace fnmoe {
namespace {

constexpr float kTiny = 0x1p-100f;   // least magnitude a scale is made for
constexpr uint32_t kMaxDim = 16384;  // columns that 512 threads hold at 4 x 8 each
constexpr uint32_t kInfBits = 0x7F800000u;

struct NormView {
  const void *x, *res, *w;
  void *y, *res_out;
  uint8_t *codes;
  float *scales;
  uint64_t x_stride, res_stride;
  int64_t rows;
  int dim;
  float eps, offset;  // offset: 1 where the weight is kept as w - 1
  bool w_f32, w_vec, norm, e4m3;  // w_vec: the weight starts on a 16-byte boundary
};

// How a row's values are dealt to its G threads, 8 to a thread's chunk:
//   kEven  columns 8 q .. + 7 of chunk q, in 16-byte accesses: rows and widths on
//          boundaries of 8 values;
//   kFlat  the same over the rows laid end to end, for rows of any width that
//          are contiguous: chunk q starts on the boundary of 8 at or below the
//          row's start, chunks that reach into a neighbour's row are masked;
//   kOdd   columns (8 c + e) G + t, one value at a time: any stride and start.
enum Deal { kEven, kFlat, kOdd };

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<uint16_t>(uint16_t v) { return bf16_to_f32(v); }
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ uint16_t narrow<uint16_t>(float v) { return f32_to_bf16(v); }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// 8 adjacent values to a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_eight(T *to, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4 *>(to) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  } else {
    reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Codes of four values whose magnitudes are at most 127 (448): int8 by adding
// 1.5 2^23, whose last bit is 1, so that the sum's low byte is the nearest whole
// number (ties to even) in two's complement.
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, bool e4m3) {
  if (e4m3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
  constexpr float kWhole = 0x1.8p23f;
  const uint32_t ab = __byte_perm(__float_as_uint(__fadd_rn(a, kWhole)), __float_as_uint(__fadd_rn(b, kWhole)), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(__fadd_rn(c, kWhole)), __float_as_uint(__fadd_rn(d, kWhole)), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

// A row's values and where this thread's chunks of them lie.
struct RowAt {
  int64_t row;
  int skew;  // kFlat: values before the row in its first chunk
};
struct Columns {
  int G, t, dim;
  int64_t total;  // values of all rows
  template <Deal D>
  __device__ __forceinline__ RowAt at(int64_t row) const {
    return RowAt{row, D == kFlat ? static_cast<int>(static_cast<uint64_t>(row) * static_cast<uint32_t>(dim) & 7u) : 0};
  }
  // the column of value e of chunk c; below 0 or from dim on where there is none
  template <Deal D>
  __device__ __forceinline__ int column(const RowAt &r, int c, int e) const {
    return D == kOdd ? (c * 8 + e) * G + t : (c * G + t) * 8 + e - r.skew;
  }
  // whether chunk c lies in the row whole; whether any of it does
  template <Deal D>
  __device__ __forceinline__ bool whole(const RowAt &r, int c) const {
    const int first = column<D>(r, c, 0);
    return first >= 0 && first + 8 <= dim;
  }
  template <Deal D>
  __device__ __forceinline__ bool some(const RowAt &r, int c) const { return column<D>(r, c, 0) < dim; }
};

// 8 values as they were loaded.
template <Deal D, typename T>
struct Raw8 {
  union {
    uint4 q[sizeof(T) / 2];
    T v[8];
  };
  __device__ __forceinline__ void load(const T *x, uint64_t stride, const Columns &k, const RowAt &r, int c) {
    const T *row = x + r.row * stride;
    if constexpr (D == kOdd) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = k.column<D>(r, c, e);
        v[e] = at < k.dim ? row[at] : T(0);
      }
    } else {
      const int first = k.column<D>(r, c, 0);
      if (first < k.dim && (D == kEven || r.row * k.dim + first + 8 <= k.total)) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) q[i] = reinterpret_cast<const uint4 *>(row + first)[i];
      } else {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (D == kFlat) {  // the last values of all
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (first + e < k.dim) put(e, row[first + e]);
        }
      }
      if constexpr (D == kFlat) {
        if (!k.whole<D>(r, c)) {  // a neighbour's values do not count
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (first + e < 0 || first + e >= k.dim) put(e, T(0));
        }
      }
    }
  }
  __device__ __forceinline__ void put(int e, T x) {
    uint32_t *w = &q[sizeof(T) == 2 ? 0 : e / 4].x;
    if constexpr (sizeof(T) == 4) {
      w[e % 4] = __float_as_uint(x);
    } else {
      w[e / 2] = (e & 1) ? (w[e / 2] & 0xFFFFu) | (static_cast<uint32_t>(x) << 16) : (w[e / 2] & 0xFFFF0000u) | x;
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (D == kOdd) {
      return widen<T>(v[e]);
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t w = e < 2 ? q[0].x : e < 4 ? q[0].y : e < 6 ? q[0].z : q[0].w;
      return __uint_as_float((e & 1) ? (w & 0xFFFF0000u) : (w << 16));
    } else {
      const uint4 w = q[e / 4];
      return __uint_as_float(e % 4 == 0 ? w.x : e % 4 == 1 ? w.y : e % 4 == 2 ? w.z : w.w);
    }
  }
};

// 8 values of chunk c to contiguous rows at `to`.
template <Deal D, typename T>
__device__ __forceinline__ void store8(T *to, const Columns &k, const RowAt &r, int c, const float (&v)[8]) {
  T *row = to + r.row * k.dim;
  if (D != kOdd && k.whole<D>(r, c)) {
    store_eight(row + k.column<D>(r, c, 0), v);
  } else if (D != kEven) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = k.column<D>(r, c, e);
      if (at >= 0 && at < k.dim) row[at] = narrow<T>(v[e]);
    }
  }
}

template <Deal D>
__device__ __forceinline__ void store_codes(uint8_t *to, const Columns &k, const RowAt &r, int c, const float (&v)[8],
                                            bool bad, bool e4m3) {
  if (!k.some<D>(r, c)) return;
  uint8_t *row = to + r.row * k.dim;
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) w[h] = bad ? 0u : four_codes(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3], e4m3);
  if (D != kOdd && k.whole<D>(r, c)) {
    *reinterpret_cast<uint2 *>(row + k.column<D>(r, c, 0)) = make_uint2(w[0], w[1]);
  } else if (D != kEven) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = k.column<D>(r, c, e);
      if (at >= 0 && at < k.dim) row[at] = static_cast<uint8_t>(w[e / 4] >> (8 * (e % 4)));
    }
  }
}

// The larger of two magnitudes; not a number where either is not.
__device__ __forceinline__ float larger(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// Sum of `sum` and maximum of `top` (which is not negative) over the G threads of
// a row: a warp, or the CTA, whose warps meet in `part` (two of them in turn, so
// that one barrier is enough).
__device__ __forceinline__ void reduce_row(float &sum, float &top, int G, float2 *part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top)));
  if (G == 32) return;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(sum, top);
  __syncthreads();
  sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < G >> 5; ++i) {
    const float2 o = part[i];
    sum += o.x;
    top = larger(top, o.y);
  }
}

// Rows by G threads each: a warp (four of them a CTA) or a CTA.  TR void: no residual.
template <Deal D, int VPT, typename TX, typename TR>
__global__ void __launch_bounds__(512, VPT <= 2 ? 2 : 1) k_norm(NormView p, int G) {
  constexpr bool kRes = !std::is_void_v<TR>;
  constexpr int kAhead = VPT == 1 && D != kOdd ? 2 : 1;  // rows whose loads are under way
  using R = std::conditional_t<kRes, TR, TX>;
  __shared__ float2 part[2][16];
  extern __shared__ __align__(16) float weight[];
  const Columns k{G, static_cast<int>(threadIdx.x) % G, p.dim, p.rows * p.dim};
  const int rows_here = blockDim.x / G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows_here;
  int64_t row = static_cast<int64_t>(blockIdx.x) * rows_here + threadIdx.x / G;
  pdl_wait();
  pdl_trigger();
  Raw8<D, TX> x[kAhead][VPT];
  Raw8<D, R> r[kAhead][kRes ? VPT : 1];
  auto ask = [&](int a, int64_t at) {
    if (at >= p.rows) return;
    const RowAt ra = k.at<D>(at);
#pragma unroll
    for (int c = 0; c < VPT; ++c) x[a][c].load(static_cast<const TX *>(p.x), p.x_stride, k, ra, c);
    if constexpr (kRes) {
#pragma unroll
      for (int c = 0; c < VPT; ++c) r[a][c].load(static_cast<const R *>(p.res), p.res_stride, k, ra, c);
    }
  };
#pragma unroll
  for (int a = 0; a < kAhead; ++a) ask(a, row + a * step);
  // Weights.  kEven: a thread's columns are the same in every row, so it reads
  // them each time, from L1.  Otherwise from shared memory; kFlat: value i at
  // (i % 8) pitch + i / 8, so that threads that read value e of adjacent chunks
  // read adjacent words whatever the skew.
  const int pitch = p.dim / 8 + 1;
  auto weight_at = [&](int i) {
    return __fadd_rn(p.w_f32 ? static_cast<const float *>(p.w)[i] : bf16_to_f32(static_cast<const uint16_t *>(p.w)[i]), p.offset);
  };
  if (D != kEven && p.norm) {
    // kFlat: zeros where there is no column, which masked values are multiplied by
    const int slots = D == kFlat ? 8 * pitch : p.dim;
#pragma unroll 4
    for (int i = threadIdx.x; i < slots; i += blockDim.x)
      weight[D == kFlat ? (i & 7) * pitch + (i >> 3) : i] = i < p.dim ? weight_at(i) : 0.0f;
    if (D == kFlat && threadIdx.x == 0) weight[slots] = 0.0f;
    __syncthreads();
  }
  // this thread's weights of chunk c (where there is no value: anything, it counts as 0)
  auto weights = [&](const RowAt &ra, int c, float (&w)[8]) {
    if (!p.norm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
    } else if constexpr (D == kEven) {
      const int at = min(k.column<D>(ra, c, 0), p.dim - 8);
      if (!p.w_vec) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = weight_at(at + e);
      } else if (p.w_f32) {
        const float4 *g = reinterpret_cast<const float4 *>(static_cast<const float *>(p.w) + at);
        const float4 a = g[0], b = g[1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
      } else {
        const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.w) + at);
        const uint32_t v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __uint_as_float((e & 1) ? (v[e / 2] & 0xFFFF0000u) : (v[e / 2] << 16));
      }
      if (p.w_vec && p.offset != 0.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __fadd_rn(w[e], p.offset);
      }
    } else if constexpr (D == kFlat) {
      // (a row's last chunk may be one past dim / 8; only values before its skew count there)
      const float *at = weight + min(c * G + k.t, pitch);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = at[((e - ra.skew) & 7) * pitch - (e < ra.skew ? 1 : 0)];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weight[min(k.column<D>(ra, c, e), p.dim - 1)];
    }
  };
  const float limit = p.e4m3 ? 448.0f : 127.0f, per_dim = 1.0f / static_cast<float>(p.dim);
  int turn = 0;
  while (row < p.rows) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a, row += step) {
      if (row >= p.rows) break;  // the whole row's threads
      const RowAt ra = k.at<D>(row);
      float s[VPT][8], sum = 0.0f, top = 0.0f;
#pragma unroll
      for (int c = 0; c < VPT; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[c][e] = x[a][c].get(e);
          if constexpr (kRes) s[c][e] = __fadd_rn(s[c][e], r[a][c].get(e));
        }
      }
      ask(a, row + kAhead * step);
#pragma unroll
      for (int c = 0; c < VPT; ++c) {
        float w[8];
        weights(ra, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum = fmaf(s[c][e], s[c][e], sum);
          top = larger(top, fabsf(s[c][e] * w[e]));
        }
        if constexpr (kRes)
          if (p.res_out) store8<D>(static_cast<R *>(p.res_out), k, ra, c, s[c]);
      }
      reduce_row(sum, top, G, part[turn ^= 1]);
      float gain = 1.0f;
      if (p.norm) {
        gain = rsqrtf(fmaf(sum, per_dim, p.eps));  // to 2^-22
        // Rows whose squares or products leave float32's range (or lose bits below
        // it) are scaled by powers of two first.
        if (!(sum <= 0x1p120f) || !(top <= 0x1p125f) || sum < 0x1p-80f || top < 0x1p-60f) {
          float most = 0.0f, none = 0.0f;
#pragma unroll
          for (int c = 0; c < VPT; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(s[c][e]));
          reduce_row(none, most, G, part[turn ^= 1]);
          if (most != 0.0f && most < __uint_as_float(kInfBits)) {
            // s by 2^-e2, to between 1/4 and 1/2 at most, the root by 2^-e3, 2^e3 about
            // the larger of max |s| and sqrt(eps); s and the gain take half of
            // 2^(e2 - e3) each.  (s in two steps, since one may be no float.)
            const int e2 = ilogbf(most) + 2, e3 = p.eps > 0.0f ? max(e2, ilogbf(p.eps) / 2) : e2;
            const int of_s = (e2 - e3) / 2, by = of_s - e2;
            const float first = ldexpf(1.0f, by / 2), second = ldexpf(1.0f, by - by / 2), of_gain = ldexpf(1.0f, e2 - e3 - of_s);
            sum = 0.0f;
            top = 0.0f;
#pragma unroll
            for (int c = 0; c < VPT; ++c) {
              float w[8];
              weights(ra, c, w);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                s[c][e] *= first;
                s[c][e] *= second;
                sum = fmaf(s[c][e], s[c][e], sum);
                top = larger(top, fabsf(s[c][e] * w[e]));
              }
            }
            reduce_row(sum, top, G, part[turn ^= 1]);
            gain = rsqrtf(sum * per_dim * of_gain * of_gain + ldexpf(ldexpf(p.eps, -e3), -e3)) * of_gain;
          }
        }
      }
      float inv = 0.0f;
      bool codes_are_0 = false;
      if (p.codes) {
        const float most = top * gain, held = fmaxf(most, kTiny);
        // a row that is not finite has a scale that is not a number, and codes of 0
        const bool bad = !(top < __uint_as_float(kInfBits)) || !(most < __uint_as_float(kInfBits));
        codes_are_0 = bad;
        inv = __fdiv_rn(limit, held);
        if (k.t == 0) p.scales[row] = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(held, limit);
      }
#pragma unroll
      for (int c = 0; c < VPT; ++c) {
        float w[8];
        weights(ra, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[c][e] = s[c][e] * w[e] * gain;  // in this order none passes top gain, nor a code 127
        if (p.y) store8<D>(static_cast<TX *>(p.y), k, ra, c, s[c]);
        if (p.codes) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[c][e] *= inv;
          store_codes<D>(p.codes, k, ra, c, s[c], codes_are_0, p.e4m3);
        }
      }
    }
  }
}

// Four codes' values, whole numbers of int8 (from a byte b ^ 128 below 2^23: 2^23
// + b + 128 less that much) or e4m3 (by way of float16, exact).
__device__ __forceinline__ void four_values(uint32_t c, bool e4m3, float *v) {
  if (e4m3) {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(lo) : "h"(static_cast<uint16_t>(c)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(hi) : "h"(static_cast<uint16_t>(c >> 16)));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    c ^= 0x80808080u;
    constexpr uint32_t kSelect[4] = {0x7440, 0x7441, 0x7442, 0x7443};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(__byte_perm(c, 0x4B000000u, kSelect[e])) - (0x1p23f + 128.0f);
  }
}

// Values of codes, 16 adjacent ones a thread whatever rows they lie in (codes
// and values are contiguous), the last few one by one.  VEC: both start on
// 16-byte boundaries.  Bound by HBM's latency: 5000 x 2048 to bfloat16 about 8 us
// (31 MB); one code a thread took 50 us at 5003 x 2561.
template <bool VEC, typename T>
__global__ void __launch_bounds__(256) k_dequantize_rows(const uint8_t *codes, const float *scales, T *out,
                                                         uint64_t count, uint32_t dim, bool e4m3) {
  constexpr int U = 16;
  pdl_wait();
  pdl_trigger();
  const uint64_t units = (count + U - 1) / U;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < units;
       i += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
    const uint64_t first = U * i;
    const int n = static_cast<int>(min(count - first, static_cast<uint64_t>(U)));
    const bool vec = VEC && n == U;
    uint32_t c[U / 4] = {};
    if (vec) {
      const uint4 q = *reinterpret_cast<const uint4 *>(codes + first);
      c[0] = q.x, c[1] = q.y, c[2] = q.z, c[3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (e < n) c[e / 4] |= static_cast<uint32_t>(codes[first + e]) << (8 * (e % 4));
    }
    uint64_t row = (count >> 32) ? first / dim : static_cast<uint32_t>(first) / dim;
    const uint64_t left = (row + 1) * dim - first;  // codes of this row from here on
    float v[U];
#pragma unroll
    for (int e = 0; e < U; e += 4) four_values(c[e / 4], e4m3, v + e);
    float scale = scales[row];
    if (left >= static_cast<uint64_t>(n)) {
#pragma unroll
      for (int e = 0; e < U; ++e) v[e] = __fmul_rn(v[e], scale);
    } else {
      uint32_t until = static_cast<uint32_t>(left);
#pragma unroll
      for (int e = 0; e < U; ++e) {
        if (static_cast<uint32_t>(e) == until && e < n) scale = scales[++row], until += dim;
        v[e] = __fmul_rn(v[e], scale);
      }
    }
    if (vec) {
#pragma unroll
      for (int h = 0; h < U; h += 8) {
        const float eight[8] = {v[h], v[h + 1], v[h + 2], v[h + 3], v[h + 4], v[h + 5], v[h + 6], v[h + 7]};
        store_eight(out + first + h, eight);
      }
    } else {
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (e < n) out[first + e] = narrow<T>(v[e]);
    }
  }
}

bool misaligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

// Bytes of a row's weights in shared memory (kFlat's eight columns of them and a zero; kOdd takes fewer).
constexpr int weight_smem(uint32_t dim) { return static_cast<int>(((dim / 8 + 1) * 8 + 1) * sizeof(float)); }

template <Deal D, int VPT, typename TX, typename TR>
cudaError_t launch_k(const NormView &p, int per, int G, cudaStream_t s) {
  const size_t smem = p.norm && D != kEven ? weight_smem(static_cast<uint32_t>(p.dim)) : 0;
  if (smem > 40 * 1024) {  // (48 KB with the kernel's own need no leave)
    static SmemLimit limit;
    const cudaError_t e = limit.set(reinterpret_cast<const void *>(k_norm<D, VPT, TX, TR>), weight_smem(kMaxDim));
    if (e != cudaSuccess) return e;
  }
  // as many CTAs as stay on the SMs: 1024 threads (512 where a thread holds more of a row)
  const int ctas = std::max(1, (VPT <= 2 ? 1024 : 512) / (per * G));
  const int64_t most = static_cast<int64_t>(device_info().sms) * ctas, need = (p.rows + per - 1) / per;
  return launch_pdl(k_norm<D, VPT, TX, TR>, dim3(static_cast<unsigned>(std::min(need, most))), dim3(per * G), smem, s, p, G);
}

template <Deal D, typename TX>
cudaError_t launch_norm(const NormView &p, uint32_t res_dtype, cudaStream_t s) {
  const int chunks = (p.dim + 7) / 8 + (D == kFlat && p.dim % 8 != 0 ? 1 : 0);  // a row off its boundary touches one more
  // A thread's chunks: one, so that few rows wait least for one another's sums,
  // or, from two rows an SM on, two where they fit the registers: the
  // sums' steps and the row's root and quotient cost a thread as much as a chunk.
  const bool wide = p.res && (sizeof(TX) == 4 || res_dtype == FNMOE_DTYPE_F32);
  const int many = p.rows >= 2 * device_info().sms && !wide ? 2 : 1;
  const int vpt = std::max(many, chunks > 1024 ? 4 : chunks > 512 ? 2 : 1);
  const int G = (chunks + 32 * vpt - 1) / (32 * vpt) * 32, per = G == 32 ? 4 : 1;
  auto go = [&](auto residual) {
    using TR = typename decltype(residual)::type;
    switch (vpt) {
      case 1: return launch_k<D, 1, TX, TR>(p, per, G, s);
      case 2: return launch_k<D, 2, TX, TR>(p, per, G, s);
      default: return launch_k<D, 4, TX, TR>(p, per, G, s);
    }
  };
  if (!p.res) return go(std::common_type<void>{});
  if (res_dtype == FNMOE_DTYPE_F32) return go(std::common_type<float>{});
  return go(std::common_type<uint16_t>{});
}

template <typename TX>
cudaError_t launch_deal(const NormView &p, Deal d, uint32_t res_dtype, cudaStream_t s) {
  switch (d) {
    case kEven: return launch_norm<kEven, TX>(p, res_dtype, s);
    case kFlat: return launch_norm<kFlat, TX>(p, res_dtype, s);
    default: return launch_norm<kOdd, TX>(p, res_dtype, s);
  }
}

int done(cudaError_t e, const char *what, std::string &err) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return FNMOE_OK;
  err = std::string(what) + ": " + cudaGetErrorString(e);
  return FNMOE_ERR_LAUNCH;
}

}  // namespace

int add_rms_norm(const FnNormArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  const bool norm = !(a->flags & FNMOE_NORM_ROWS_AS_THEY_ARE);
  if (a->dim == 0 || a->dim > kMaxDim) {
    err = "dim must be between 1 and " + std::to_string(kMaxDim);
    return FNMOE_ERR_SHAPE;
  }
  if (a->rows > 0x7FFFFFFFu) { err = "at most 2^31 - 1 rows"; return FNMOE_ERR_SHAPE; }
  if (a->x_dtype > FNMOE_DTYPE_F32 || a->residual_dtype > FNMOE_DTYPE_F32 || a->weight_dtype > FNMOE_DTYPE_F32 ||
      a->code_type > FNMOE_Q8_E4M3) {
    err = "x, residual and weight must be bfloat16 or float32, codes int8 or e4m3";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (norm && !(a->eps >= 0.0f && a->eps < __builtin_inff())) { err = "eps must be finite and not negative"; return FNMOE_ERR_VALUE; }
  if (a->rows == 0) return FNMOE_OK;
  if (!a->x || (norm && !a->weight)) { err = "x and weight are required"; return FNMOE_ERR_NULL; }
  if ((!a->y && !a->codes) || (a->codes && !a->scales)) {
    err = "y or codes is required, and scales with codes";
    return FNMOE_ERR_NULL;
  }
  if (a->residual_out && !a->residual) { err = "residual_out needs residual"; return FNMOE_ERR_NULL; }
  if (a->rows > 1 && (a->x_stride < a->dim || (a->residual && a->residual_stride < a->dim))) {
    err = "row strides must cover dim values";
    return FNMOE_ERR_SHAPE;
  }
  const uintptr_t xs = a->x_dtype == FNMOE_DTYPE_F32 ? 4 : 2, rs = a->residual_dtype == FNMOE_DTYPE_F32 ? 4 : 2,
                  ws = a->weight_dtype == FNMOE_DTYPE_F32 ? 4 : 2;
  if (misaligned(a->x, xs) || misaligned(a->y, xs) || misaligned(a->residual, rs) || misaligned(a->residual_out, rs) ||
      (norm && misaligned(a->weight, ws)) || misaligned(a->scales, 4)) {
    err = "arrays must be aligned to their elements";
    return FNMOE_ERR_VALUE;
  }
  const uint64_t rows = a->rows, n = rows * a->dim;
  const Span x{a->x, ((rows - 1) * a->x_stride + a->dim) * xs}, res{a->residual, ((rows - 1) * a->residual_stride + a->dim) * rs},
      w{norm ? a->weight : nullptr, a->dim * ws}, y{a->y, n * xs}, out{a->residual_out, n * rs}, codes{a->codes, n},
      scales{a->scales, rows * 4};
  // in place: the same rows in the same place
  const bool y_in_x = a->y == a->x && (rows == 1 || a->x_stride == a->dim),
             out_in_res = a->residual_out == a->residual && (rows == 1 || a->residual_stride == a->dim);
  if ((!y_in_x && y.meets(x)) || y.meets(res) || y.meets(w) || y.meets(out) || out.meets(x) || (!out_in_res && out.meets(res)) ||
      out.meets(w) || codes.meets(x) || codes.meets(res) || codes.meets(w) || codes.meets(y) || codes.meets(out) ||
      scales.meets(x) || scales.meets(res) || scales.meets(w) || scales.meets(y) || scales.meets(out) || scales.meets(codes)) {
    err = "outputs overlap inputs or one another (residual_out may be residual, y may be x, where rows are adjacent)";
    return FNMOE_ERR_VALUE;
  }
  NormView p{};
  p.x = a->x;
  p.res = a->residual;
  p.w = a->weight;
  p.y = a->y;
  p.res_out = a->residual_out;
  p.codes = static_cast<uint8_t *>(a->codes);
  p.scales = a->scales;
  p.x_stride = a->x_stride;
  p.res_stride = a->residual_stride;
  p.rows = a->rows;
  p.dim = static_cast<int>(a->dim);
  p.eps = a->eps;
  p.offset = (a->flags & FNMOE_NORM_UNIT_OFFSET) ? 1.0f : 0.0f;
  p.w_f32 = a->weight_dtype == FNMOE_DTYPE_F32;
  p.w_vec = !misaligned(a->weight, 16);
  p.norm = norm;
  p.e4m3 = a->code_type == FNMOE_Q8_E4M3;
  const bool starts = !misaligned(a->x, 16) && !misaligned(a->residual, 16) && !misaligned(a->y, 16) &&
                      !misaligned(a->residual_out, 16) && !misaligned(a->codes, 8);
  const bool even = a->dim % 8 == 0 && (a->rows == 1 || (a->x_stride * xs % 16 == 0 &&
                    (!a->residual || a->residual_stride * rs % 16 == 0)));
  const bool contiguous = a->rows == 1 || (a->x_stride == a->dim && (!a->residual || a->residual_stride == a->dim));
  // (kFlat holds up to 16376 columns: its rows may touch one chunk more)
  const Deal d = starts && even ? kEven : starts && contiguous && a->dim <= kMaxDim - 8 ? kFlat : kOdd;
  const cudaError_t e = a->x_dtype == FNMOE_DTYPE_F32 ? launch_deal<float>(p, d, a->residual_dtype, s)
                                                      : launch_deal<uint16_t>(p, d, a->residual_dtype, s);
  return done(e, "add_rms_norm", err);
}

int dequantize_rows(const FnRowCodesArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (a->dim == 0) { err = "dim must be positive"; return FNMOE_ERR_SHAPE; }
  if (a->code_type > FNMOE_Q8_E4M3 || a->out_dtype > FNMOE_DTYPE_F32) {
    err = "codes must be int8 or e4m3, out bfloat16 or float32";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (a->rows == 0) return FNMOE_OK;
  if (!a->codes || !a->scales || !a->out) { err = "codes, scales and out are required"; return FNMOE_ERR_NULL; }
  const bool f32 = a->out_dtype == FNMOE_DTYPE_F32, e4m3 = a->code_type == FNMOE_Q8_E4M3;
  if (misaligned(a->scales, 4) || misaligned(a->out, f32 ? 4 : 2)) {
    err = "scales and out must be aligned to their elements";
    return FNMOE_ERR_VALUE;
  }
  const uint64_t count = static_cast<uint64_t>(a->rows) * a->dim;
  const Span out{a->out, count * (f32 ? 4 : 2)};
  if (out.meets(Span{a->codes, count}) || out.meets(Span{a->scales, static_cast<uint64_t>(a->rows) * 4})) {
    err = "out overlaps codes or scales";
    return FNMOE_ERR_VALUE;
  }
  const bool vec = !misaligned(a->codes, 16) && !misaligned(a->out, 16);
  const dim3 grid(static_cast<unsigned>(std::min<uint64_t>((count + 4095) / 4096, 1u << 20)));
  const uint8_t *c = static_cast<const uint8_t *>(a->codes);
  cudaError_t e;
  if (f32) {
    float *o = static_cast<float *>(a->out);
    e = vec ? launch_pdl(k_dequantize_rows<true, float>, grid, dim3(256), 0, s, c, a->scales, o, count, a->dim, e4m3)
            : launch_pdl(k_dequantize_rows<false, float>, grid, dim3(256), 0, s, c, a->scales, o, count, a->dim, e4m3);
  } else {
    uint16_t *o = static_cast<uint16_t *>(a->out);
    e = vec ? launch_pdl(k_dequantize_rows<true, uint16_t>, grid, dim3(256), 0, s, c, a->scales, o, count, a->dim, e4m3)
            : launch_pdl(k_dequantize_rows<false, uint16_t>, grid, dim3(256), 0, s, c, a->scales, o, count, a->dim, e4m3);
  }
  return done(e, "dequantize_rows", err);
}

}  // namespace fnmoe
