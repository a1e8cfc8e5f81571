// attention_q8.cuh -- what the kernels of the attention over the paged 8-bit
// KV cache share: the call's view, code conversion, the row and token counts
// of a sequence and the division of work.
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale * q_i . k_j - m_i),
//   k_j = ks[block of j] * kcode_j,  v_j = vs[block of j] * vcode_j,
//   j over the positions up to row i's own whose page is in the cache.
//
// Codes go to the tensor cores as numbers in which they are exact (bfloat16
// holds int8's 7 bits and sign and e4m3's 4 bits); the two block scales enter
// in float32.  With
//   t_j = (scale * log2 e * ks) (q . kcode_j) + log2 vs,   u_j = 2^(t_j - m),
// m a running reference of the t_j,
//   out = sum_j u_j vcode_j / sum_blocks (1 / vs) sum_(j in block) u_j :
// the value scale rides in the exponent.  The sums hold t_j within 2^126 of the
// reference, so a block whose vs is far below its neighbours' would drop out of
// the denominator, where its tokens count in full whatever their values: a block
// of zeros has vs = 2^-107.  Its vs is therefore raised to vs' = 2^-64 of the
// largest that the warp (or tile) has met in its piece of work, which leaves
// weights down to 2^-62 of the largest in the denominator, and its weights go
// into the second product as u_j vs / vs', at least 2^-62 of the largest weight
// where the scales lie within 2^128 of each other; beyond that the values of the
// smaller blocks fade.  vs' is at least 2^-90, so that no denominator overflows.
//   The weights enter the second product
// as two bfloat16 terms, u = hi + lo with 16 bits: one term alone would cost
// up to 2^-9 of an output (as much as its final rounding), and float16 loses
// weights below 2^-24 of the largest, which are all that is left of an output
// whose heaviest tokens hold zeros.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "async.cuh"
#include "common.cuh"
#include "q8_ranges.cuh"

namespace fnmoe {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;  // a reference may fall this far (log2) below the largest t
constexpr float kScaleSpan = 0x1p-64f, kScaleLeast = 0x1p-90f;  // vs' >= vs of the largest block * span, and >= least

constexpr int kUnit = 64;  // tokens of a unit of work

struct Q8View {
  const uint16_t *q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *ctx, *cu;
  uint16_t *out;
  uint64_t q_stride;
  int B, rows, Hq, Hkv, gq, page, block_shift, width, pages;
  uint32_t page_magic;  // 2^32 / page, rounded up
  float scale;
  int few_rows;         // sequences of more (row, head) pairs per kv head take the many-row kernel
  // workspace of the few-row kernel (8 rows a tile)
  int4 *cuts;           // [CTAs] where each range begins (cut_of), or by_seg: [B][Hkv][few_tiles]
  int few_tiles;        // tiles of 8 rows that a sequence can have
  int join_rows;        // rows that such a tile can have
  int ctas, tctas;      // CTAs of the few-row and the many-row kernel
  bool by_seg, tby_seg, pair_boxes;
  float *part;          // [2 * CTAs][8][D] unfinished sums
  float2 *part_ml;      // [2 * CTAs][8] their reference and weight sum
  // workspace of the many-row kernel (128 rows a tile)
  int max_tiles;
  int *seq_tile;        // [B + 1] tiles before each sequence
  int4 *tiles;          // [tiles] {sequence, tile of it, units of one kv head, 0}
  int4 *tcuts;          // [CTAs], or tby_seg: [tiles][Hkv]
  long long *tprefix;   // [tiles + 1] units of work before each tile
  float *tpart;         // [2 * CTAs][D / 4][128][4]
  float2 *tpart_ml;     // [2 * CTAs][128]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// Of normal numbers; within 2^-22 and 2^-23.
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// x 2^d where 2^d alone may be too small for a float: a denominator's sum can be
// as large as 2^90 of its weights.
__device__ __forceinline__ float times_ex2(float x, float d) {
  const float h = ex2(0.5f * d);
  return x * h * h;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;\n" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two float32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n"
      : "=l"(d)
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
        "l"(reinterpret_cast<unsigned long long &>(c)));
  return reinterpret_cast<float2 &>(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;\n"
      : "=l"(d)
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return reinterpret_cast<float2 &>(d);
}
// a and b as bfloat16 pairs hi + lo.
__device__ __forceinline__ void split_bf16x2(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = pack_bf16x2(a, b);
  lo = pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
}
__device__ __forceinline__ void mma_bf16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// m16n8k32 with signed A bytes and unsigned (or signed) B bytes.
template <bool SIGNED_B>
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (SIGNED_B)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two e4m3 codes in bytes (0, 1) or (2, 3) of w as float16.
template <int HALF>
__device__ __forceinline__ uint32_t e4m3_f16(uint32_t w) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(static_cast<uint16_t>(HALF ? w >> 16 : w)));
  return h;
}

// Two codes in bytes (0, 1) (HALF 0) or (2, 3) (HALF 1) of w, as bfloat16 pairs.
// int8: under the high byte 0x43, the low seven bits l of a code read as
// 128 + l and its sign bit alone as 128 (clear) or 256 (set); the difference
// is l or l - 128, the code.
// e4m3: to float16, to float32, to bfloat16, all exact.
template <bool E4M3, int HALF>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  uint32_t d;
  if (E4M3) {
    const uint32_t h = e4m3_f16<HALF>(w);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    d = pack_bf16x2(f.x, f.y);
  } else {
    const uint32_t x = prmt(w, 0x43434343u, HALF ? 0x4342u : 0x4140u);
    asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(x & 0xFF7FFF7Fu), "r"(x & 0xFF80FF80u));
  }
  return d;
}

// Codes of four dims of two tokens (words w0, w1) as bfloat16 pairs (token 0,
// token 1), one for each dim.  int8 as in widen2, with the byte that prmt
// leaves between the two replaced under the mask.
template <bool E4M3>
__device__ __forceinline__ void widen_pairs(uint32_t w0, uint32_t w1, uint32_t (&d)[4]) {
  if (E4M3) {
    const uint32_t lo = prmt(w0, w1, 0x5140u), hi = prmt(w0, w1, 0x7362u);
    d[0] = widen2<true, 0>(lo);
    d[1] = widen2<true, 1>(lo);
    d[2] = widen2<true, 0>(hi);
    d[3] = widen2<true, 1>(hi);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t x = prmt(w0, w1, i | (i << 4) | ((4 + i) << 8) | ((4 + i) << 12));
      uint32_t a, b;  // (x & mask) | 0x43004300
      asm("lop3.b32 %0, %1, 0x007F007F, 0x43004300, 0xEA;\n" : "=r"(a) : "r"(x));
      asm("lop3.b32 %0, %1, 0x00800080, 0x43004300, 0xEA;\n" : "=r"(b) : "r"(x));
      asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(d[i]) : "r"(a), "r"(b));
    }
  }
}

// 16 bytes, read once by this CTA.  The kernels may be resident while an earlier one of the
// stream still writes (programmatic dependent launch), so nothing that such a
// kernel produced -- queries, codes, scales -- is read through the non-coherent
// path.  (Past L1 altogether, ld.global.cg: prefill chunk 356 us instead of 375,
// 16 sequences of verify rows 101 instead of 89.)
__device__ __forceinline__ uint4 ldg_stream(const void *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Rows of sequence b: first packed row and their number.
__device__ __forceinline__ int2 rows_of(const Q8View &p, int b) {
  if (p.cu == nullptr) return make_int2(b, 1);
  const int r0 = max(p.cu[b], 0), r1 = min(p.cu[b + 1], p.rows);
  return make_int2(r0, max(r1 - r0, 0));
}
// pos / page for pos < 2^31.
__device__ __forceinline__ int page_col(const Q8View &p, int pos) {
  int c = static_cast<int>(__umulhi(static_cast<uint32_t>(pos), p.page_magic));
  if (c * p.page > pos) --c;
  return c;
}
// Tokens of sequence b that the cache can hold.
__device__ __forceinline__ int tokens_of(const Q8View &p, int b) {
  return max(0, min(p.ctx[b], p.width * p.page));
}

// The many-row kernels (attention_q8_many.cu).
int many_ctas(int head_dim);
uint64_t many_tiles(const Q8View &p);  // at most so many tiles of 128 rows
int few_ctas(int head_dim);
cudaError_t launch_many(const Q8View &p, int head_dim, bool e4m3, cudaStream_t s);

}  // namespace fnmoe
