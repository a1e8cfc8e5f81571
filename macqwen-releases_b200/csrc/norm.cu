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
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "dense.cuh"

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
  bool w_f32, norm, e4m3;
};

// 8 values of a row.  VEC: columns 8 (c G + t) .. + 7 in one or two 16-byte
// accesses; else columns (8 c + e) G + t, one by one but coalesced.
template <bool VEC>
__device__ __forceinline__ int column(int c, int e, int G, int t) {
  return VEC ? (c * G + t) * 8 + e : (c * 8 + e) * G + t;
}

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

template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T *row, int c, int G, int t, int dim, float (&v)[8]) {
  if constexpr (VEC) {
    const int at = column<true>(c, 0, G, t);
    if (at >= dim) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    } else if constexpr (sizeof(T) == 2) {
      const uint4 q = *reinterpret_cast<const uint4 *>(row + at);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float((e & 1) ? (w[e / 2] & 0xFFFF0000u) : (w[e / 2] << 16));
    } else {
      const float4 a = *reinterpret_cast<const float4 *>(row + at), b = *reinterpret_cast<const float4 *>(row + at + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = column<false>(c, e, G, t);
      v[e] = at < dim ? widen<T>(row[at]) : 0.0f;
    }
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T *row, int c, int G, int t, int dim, const float (&v)[8]) {
  if constexpr (VEC) {
    const int at = column<true>(c, 0, G, t);
    if (at >= dim) return;
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = static_cast<uint32_t>(f32_to_bf16(v[2 * e])) | (static_cast<uint32_t>(f32_to_bf16(v[2 * e + 1])) << 16);
      *reinterpret_cast<uint4 *>(row + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<float4 *>(row + at) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4 *>(row + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = column<false>(c, e, G, t);
      if (at < dim) row[at] = narrow<T>(v[e]);
    }
  }
}

__device__ __forceinline__ uint8_t code_of(float v, bool e4m3) {
  if (e4m3) return static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3));
  return static_cast<uint8_t>(max(-127, min(127, __float2int_rn(v))));
}

template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t *row, int c, int G, int t, int dim, const float (&v)[8], bool e4m3) {
  if constexpr (VEC) {
    const int at = column<true>(c, 0, G, t);
    if (at >= dim) return;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= static_cast<uint32_t>(code_of(v[e], e4m3)) << (8 * (e & 3));
    *reinterpret_cast<uint2 *>(row + at) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = column<false>(c, e, G, t);
      if (at < dim) row[at] = code_of(v[e], e4m3);
    }
  }
}

// Sum of `sum` and maximum of `top` over the G threads of a row (all threads
// of the CTA call it together; `part` has two words a warp).
__device__ __forceinline__ void reduce_row(float &sum, uint32_t &top, int G, float2 *part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (G == 32) return;
  const int warp = threadIdx.x >> 5, per = G >> 5, first = warp / per * per;
  __syncthreads();  // a second reduction does not overtake the first one's reads
  if ((threadIdx.x & 31) == 0) part[warp] = make_float2(sum, __uint_as_float(top));
  __syncthreads();
  sum = 0.0f;
  top = 0u;
  for (int i = first; i < first + per; ++i) {
    sum += part[i].x;
    top = max(top, __float_as_uint(part[i].y));
  }
}

// One row per G threads; a CTA holds blockDim.x / G rows.  TR void: no residual.
template <bool VEC, int VPT, typename TX, typename TR>
__global__ void __launch_bounds__(512) k_norm(NormView p, int G) {
  __shared__ float2 part[16];
  const int t = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / G) + threadIdx.x / G;
  const bool live = row < p.rows;  // threads past the last row only keep the barriers company
  pdl_wait();
  pdl_trigger();
  float s[VPT][8];
#pragma unroll
  for (int c = 0; c < VPT; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[c][e] = 0.0f;
  if (live) {
    const TX *x = static_cast<const TX *>(p.x) + row * p.x_stride;
#pragma unroll
    for (int c = 0; c < VPT; ++c) load8<VEC>(x, c, G, t, p.dim, s[c]);
    if constexpr (!std::is_void_v<TR>) {
      const TR *r = static_cast<const TR *>(p.res) + row * p.res_stride;
      float add[VPT][8];
#pragma unroll
      for (int c = 0; c < VPT; ++c) load8<VEC>(r, c, G, t, p.dim, add[c]);
#pragma unroll
      for (int c = 0; c < VPT; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[c][e] = __fadd_rn(s[c][e], add[c][e]);
        if (p.res_out) store8<VEC>(static_cast<TR *>(p.res_out) + row * p.dim, c, G, t, p.dim, s[c]);
      }
    }
  }
  float sum = 0.0f, w[VPT][8];
  uint32_t top = 0u;
#pragma unroll
  for (int c = 0; c < VPT; ++c) {
    if (p.norm && live) {
      if (p.w_f32) load8<VEC>(static_cast<const float *>(p.w), c, G, t, p.dim, w[c]);
      else load8<VEC>(static_cast<const uint16_t *>(p.w), c, G, t, p.dim, w[c]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[c][e] = p.norm && live ? __fadd_rn(w[c][e], p.offset) : 1.0f;
      sum = fmaf(s[c][e], s[c][e], sum);
      top = max(top, __float_as_uint(s[c][e] * w[c][e]) & 0x7FFFFFFFu);
    }
  }
  reduce_row(sum, top, G, part);
  float gain = 1.0f;
  if (p.norm) {
    const float n = static_cast<float>(p.dim);
    // Rows whose squares or products leave float32's range (or lose bits below
    // it) are scaled by a power of two first.  Every thread of the CTA takes
    // part, so that rows that share a CTA may differ.
    const bool far = !(sum <= 0x1p120f) || top > 0x7E000000u || (sum < 0x1p-80f && p.eps < 0x1p-80f);
    float rms_eps = p.eps;
    if (__syncthreads_or(far)) {
      uint32_t most = 0u;
      float none = 0.0f;
#pragma unroll
      for (int c = 0; c < VPT; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(s[c][e]) & 0x7FFFFFFFu);
      reduce_row(none, most, G, part);
      // by 2^-e with 2^e about the larger of max |s| and sqrt(eps); by 1 where that is 0 or not finite
      int e2 = 0;
      if (far && most != 0u && most < kInfBits) {
        e2 = max(-126, min(126, ilogbf(__uint_as_float(most))));
        if (p.eps > 0.0f) e2 = max(e2, ilogbf(p.eps) / 2);
      }
      const float down = ldexpf(1.0f, -e2);
      rms_eps = ldexpf(ldexpf(p.eps, -e2), -e2);
      sum = 0.0f;
      top = 0u;
#pragma unroll
      for (int c = 0; c < VPT; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[c][e] *= down;
          sum = fmaf(s[c][e], s[c][e], sum);
          top = max(top, __float_as_uint(s[c][e] * w[c][e]) & 0x7FFFFFFFu);
        }
      reduce_row(sum, top, G, part);
    }
    gain = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, n), rms_eps)));
  }
  if (!live) return;
#pragma unroll
  for (int c = 0; c < VPT; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[c][e] = s[c][e] * gain * w[c][e];
  if (p.y)
#pragma unroll
    for (int c = 0; c < VPT; ++c) store8<VEC>(static_cast<TX *>(p.y) + row * p.dim, c, G, t, p.dim, s[c]);
  if (p.codes) {
    const float limit = p.e4m3 ? 448.0f : 127.0f;
    const float most = __uint_as_float(top) * gain;
    // a row that is not finite has a scale that is not a number, and codes of 0
    const bool bad = !(most < __uint_as_float(kInfBits));
    const float held = fmaxf(most, kTiny);
    const float inv = bad ? 0.0f : __fdiv_rn(limit, held);
    if (t == 0) p.scales[row] = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(held, limit);
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] = bad ? 0.0f : s[c][e] * inv;
      store_codes<VEC>(p.codes + row * p.dim, c, G, t, p.dim, s[c], p.e4m3);
    }
  }
}

// Values of codes: a unit of U codes (one access) per thread.
template <int U, typename T>
__global__ void __launch_bounds__(256) k_dequantize_rows(const uint8_t *codes, const float *scales, T *out,
                                                         uint64_t units, uint32_t per_row, bool e4m3) {
  pdl_wait();
  pdl_trigger();
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < units;
       i += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
    const uint64_t row = (units >> 32) ? i / per_row : static_cast<uint32_t>(i) / per_row;
    const float scale = scales[row];
    uint8_t c[U];
    if constexpr (U == 8) *reinterpret_cast<uint2 *>(c) = *reinterpret_cast<const uint2 *>(codes + 8 * i);
    else c[0] = codes[i];
    float v[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const float q = e4m3 ? __half2float(__nv_cvt_fp8_to_halfraw(c[e], __NV_E4M3))
                           : static_cast<float>(static_cast<int8_t>(c[e]));
      v[e] = __fmul_rn(q, scale);
    }
    if constexpr (U == 8) store8<true>(out + 8 * i, 0, 1, 0, 8, v);
    else out[i] = narrow<T>(v[0]);
  }
}

bool misaligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <bool VEC, int VPT, typename TX>
cudaError_t launch_res(const NormView &p, uint32_t res_dtype, dim3 grid, int threads, int G, cudaStream_t s) {
  if (!p.res) return launch_pdl(k_norm<VEC, VPT, TX, void>, grid, dim3(threads), 0, s, p, G);
  if (res_dtype == FNMOE_DTYPE_F32) return launch_pdl(k_norm<VEC, VPT, TX, float>, grid, dim3(threads), 0, s, p, G);
  return launch_pdl(k_norm<VEC, VPT, TX, uint16_t>, grid, dim3(threads), 0, s, p, G);
}

template <bool VEC, typename TX>
cudaError_t launch_norm(const NormView &p, uint32_t res_dtype, cudaStream_t s) {
  const int chunks = (p.dim + 7) / 8;
  int vpt = chunks > 1024 ? 4 : chunks > 512 ? 2 : 1;
  const int G = (chunks + 32 * vpt - 1) / (32 * vpt) * 32;
  const int per = std::max(1, 128 / G);  // rows of a CTA
  const dim3 grid(static_cast<unsigned>((p.rows + per - 1) / per));
  switch (vpt) {
    case 1: return launch_res<VEC, 1, TX>(p, res_dtype, grid, per * G, G, s);
    case 2: return launch_res<VEC, 2, TX>(p, res_dtype, grid, per * G, G, s);
    default: return launch_res<VEC, 4, TX>(p, res_dtype, grid, per * G, G, s);
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
  p.norm = norm;
  p.e4m3 = a->code_type == FNMOE_Q8_E4M3;
  // 16-byte accesses where every row of every array allows them
  const bool vec = a->dim % 8 == 0 && !misaligned(a->x, 16) && !misaligned(a->residual, 16) &&
                   !(norm && misaligned(a->weight, 16)) && !misaligned(a->y, 16) && !misaligned(a->residual_out, 16) &&
                   !misaligned(a->codes, 8) && (a->rows == 1 || (a->x_stride * xs % 16 == 0 &&
                   (!a->residual || a->residual_stride * rs % 16 == 0)));
  cudaError_t e;
  if (a->x_dtype == FNMOE_DTYPE_F32) e = vec ? launch_norm<true, float>(p, a->residual_dtype, s) : launch_norm<false, float>(p, a->residual_dtype, s);
  else e = vec ? launch_norm<true, uint16_t>(p, a->residual_dtype, s) : launch_norm<false, uint16_t>(p, a->residual_dtype, s);
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
  const bool vec = a->dim % 8 == 0 && !misaligned(a->codes, 8) && !misaligned(a->out, 16);
  const uint32_t per_row = vec ? a->dim / 8 : a->dim;
  const uint64_t units = static_cast<uint64_t>(a->rows) * per_row;
  const dim3 grid(static_cast<unsigned>(std::min<uint64_t>((units + 255) / 256, 1u << 20)));
  const uint8_t *c = static_cast<const uint8_t *>(a->codes);
  cudaError_t e;
  if (f32) {
    float *o = static_cast<float *>(a->out);
    e = vec ? launch_pdl(k_dequantize_rows<8, float>, grid, dim3(256), 0, s, c, a->scales, o, units, per_row, e4m3)
            : launch_pdl(k_dequantize_rows<1, float>, grid, dim3(256), 0, s, c, a->scales, o, units, per_row, e4m3);
  } else {
    uint16_t *o = static_cast<uint16_t *>(a->out);
    e = vec ? launch_pdl(k_dequantize_rows<8, uint16_t>, grid, dim3(256), 0, s, c, a->scales, o, units, per_row, e4m3)
            : launch_pdl(k_dequantize_rows<1, uint16_t>, grid, dim3(256), 0, s, c, a->scales, o, units, per_row, e4m3);
  }
  return done(e, "dequantize_rows", err);
}

}  // namespace fnmoe
