// linear.cu -- out = act(x_scale weight_scale (x weight^T) + bias) + residual
// for bfloat16 rows and weights, or 8-bit ones (int8, e4m3) with a scale a row.
//
// tcgen05 with the operands' roles exchanged: 128 weight rows are the MMA's M
// (TMEM lanes), 16 to 256 rows of x its N (TMEM columns).  A decode step of a
// few rows then pads x to 16 columns instead of 128 rows, the weight's stream
// is one 16 KB TMA box a k-step whatever the batch, and a lane's bias and
// weight scale are one register.  A k-step is 128 bytes of both operands' rows
// (128-byte swizzle); the ring's boxes are zero past the matrices' ends, so
// ragged sizes need no masks before the stores.
//
// Sums: float32 in TMEM for bfloat16 and e4m3, exact int32 for int8 (widths up
// to 131071 keep 128^2 K below 2^31).  The epilogue works on float32 and rounds
// once, to the output's type.
//
// Measured: 16 x 2048 > 131072 (a head) 88 us, 6.2 TB/s; 1 x 2048 > 5120 7.9 us;
// 5000 x 2048 > 5120 with SiLU 84 us, 1,248 TFLOP/s of 1,653, with pauses between
// the calls (98 us back to back, under the power limit); 8192 x 4096 x 4096 int8
// 95 us, 2,890 TOPS.
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>

#include "async.cuh"
#include "common.cuh"
#include "dense.cuh"
#include "moe_kernels.cuh"
#include "umma.cuh"

namespace fnmoe {
namespace {

constexpr int kLanes = 128;            // weight rows of a tile
constexpr int kBoxW = kLanes * 128;    // bytes of a k-step's weight box
constexpr uint32_t kSpin = 1u << 20;   // polls before a wait gives up
constexpr uint32_t kMaxWidth = 131071;

enum Kind { kBf16 = FNMOE_LINEAR_BF16, kInt8 = FNMOE_LINEAR_INT8, kE4m3 = FNMOE_LINEAR_E4M3 };

struct LinearView {
  const float *xs, *ws;
  const void *bias, *res;
  void *out;
  uint64_t res_stride;
  int rows, width, k_steps;  // rows of x, columns of out, k-steps of 128 bytes
  int tile;                  // rows of x in an item: a multiple of 16, at most the kernel's NT
  int x_tiles, items;
  int split;                 // CTAs of a cluster that share an item's k-steps
  int chunk;                 // k-steps that are summed in TMEM at once
  uint32_t act;
  bool bias_f32, res_f32, out_f32;
  bool xs_vec;               // xs starts on a 16-byte boundary
};

// NT: most rows of x in an item.  PAIR: two CTAs with 128 weight rows each share
// an item's rows of x, half of them in either's shared memory.
template <int NT, bool PAIR>
struct Shape {
  static constexpr int kBoxX = (PAIR ? NT / 2 : NT) * 128;
  static constexpr int kStage = kBoxW + kBoxX;
  // small tiles leave room for a second CTA on the SM
  static constexpr int kStages = PAIR ? 6 : NT <= 32 ? 5 : NT <= 64 ? 4 : NT <= 128 ? 6 : 4;
  static constexpr int kCtas = NT <= 64 ? 2 : 1;
  static constexpr int kEpi = NT <= 32 ? 4 : NT <= 128 ? 8 : 16;  // epilogue warps
  // sums of several chunks: at 256 columns they would not fit the registers
  static constexpr bool kSums = NT < 256;
  static constexpr int kRows = kEpi == 16 ? 8 : 16;      // rows that an epilogue thread finishes at once
  static constexpr int kThreads = 64 + 32 * kEpi;
  static constexpr int kCols = NT / (kEpi / 4);          // TMEM columns an epilogue warp reads
  static constexpr int kBarOff = kStages * kStage;
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + 2,
                       kBars = kAccEmpty + 2;
  static constexpr int kSmem = kBarOff + 8 * kBars + 16 + 1024;  // + TMEM slot, dead flag, 1 KiB alignment
  static constexpr uint32_t kTmemCols = 2 * NT < 32 ? 32 : 2 * NT > 256 ? 512 : 2 * NT;  // a power of two
  static_assert(kCtas * (kSmem + 1024) <= 227 * 1024, "shared memory");
  static_assert(PAIR || NT * kLanes * 4 <= kBarOff, "a split's partial sums lie in the ring");
};

// Instruction descriptor: D float32 (s32 for int8), both operands K-major,
// N columns, M = 128 (256 over a pair); operand formats bf16, signed 8-bit or e4m3.
template <int KIND, bool PAIR>
__device__ __forceinline__ uint32_t idesc(int n) {
  const uint32_t d = KIND == kInt8 ? 2u : 1u, ab = KIND == kE4m3 ? 0u : 1u;
  return (d << 4) | (ab << 7) | (ab << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>((PAIR ? 2 * kLanes : kLanes) >> 4) << 24);
}

#define FNMOE_MMA(GROUP, KIND_NAME)                                                                       \
  asm volatile(                                                                                           \
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"                                                      \
      " tcgen05.mma.cta_group::" GROUP ".kind::" KIND_NAME " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),         \
      "l"(a), "l"(b), "r"(id), "r"(accumulate)                                                            \
      : "memory")
template <int KIND, bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  if constexpr (PAIR) {
    if constexpr (KIND == kBf16) FNMOE_MMA("2", "f16");
    else if constexpr (KIND == kInt8) FNMOE_MMA("2", "i8");
    else FNMOE_MMA("2", "f8f6f4");
  } else {
    if constexpr (KIND == kBf16) FNMOE_MMA("1", "f16");
    else if constexpr (KIND == kInt8) FNMOE_MMA("1", "i8");
    else FNMOE_MMA("1", "f8f6f4");
  }
}
#undef FNMOE_MMA

// Arrival of the MMAs so far on `bar`; in a pair on both CTAs' (the same place in either).
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    umma_commit(bar);
}

// The cluster address of this CTA's shared address `a` in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_rank(uint32_t a, uint32_t rank) {
  uint32_t v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(v) : "r"(a), "r"(rank));
  return v;
}
__device__ __forceinline__ void arrive_in_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// A TMA box into this CTA's shared memory, completing on a barrier of the pair (a cluster address).
__device__ __forceinline__ void tma_box2d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, volatile uint32_t *dead, uint32_t *err) {
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The word at shared address `a` of this CTA, in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t peer_word(uint32_t a, uint32_t rank) {
  uint32_t v;
  asm volatile("{\n .reg .b32 p;\n mapa.shared::cluster.u32 p, %1, %2;\n ld.shared::cluster.u32 %0, [p];\n}\n"
               : "=r"(v)
               : "r"(a), "r"(rank)
               : "memory");
  return v;
}

// Activations of U values, the choice made once for all of them.  Where the
// result stays float32, by CUDA's exp and erfc.  Where it is rounded to bfloat16
// (2^-8) by the approximate exponential and quotient (2^-21) and, for GELU, by
// erfc(z) = exp(-z^2) (c1 t + .. + c6 t^6), t = 1 / (1 + 0.41 z): a tile's
// epilogue has to stay shorter than its MMAs.  The coefficients are a minimax fit
// (linear programme over 1,900 points of [0, 9.6]) to the lesser of an absolute
// and a relative error: at most 1e-7, and 2^-12 of the value as far as bfloat16
// reaches (-13).  Five terms of that absolute error alone were 0.4% off at -6.
template <int U>
__device__ __forceinline__ void activate(float (&v)[U], uint32_t act, bool f32) {
  switch (act) {
    case FNMOE_ACT_SILU:
      if (f32) {
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = __fdiv_rn(v[i], 1.0f + expf(-v[i]));
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = __fdividef(v[i], 1.0f + __expf(-v[i]));
      }
      break;
    case FNMOE_ACT_GELU:
      if (f32) {
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = 0.5f * v[i] * erfcf(-0.70710678118654752f * v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          // max(v, 0) - |v| erfc(|v| / sqrt 2) / 2; beyond 20 the second term is 0
          const float m = fminf(fabsf(v[i]), 20.0f);
          const float t = __fdividef(1.0f, fmaf(0.41f * 0.70710678f, m, 1.0f));
          float q = fmaf(-0.179154054f, t, 0.575672936f);
          q = fmaf(fmaf(fmaf(fmaf(q, t, -0.194078793f), t, 0.363653735f), t, 0.20013245f), t, 0.233773632f);
          q = q * t * __expf(-0.5f * m * m);
          v[i] = (v[i] > 0.0f ? v[i] : 0.0f * v[i]) - 0.5f * m * q;  // 0 * v: NaN stays
        }
      }
      break;
    case FNMOE_ACT_RELU:
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
      break;
    default: break;
  }
}

// This lane's part of out's rows: everything that depends on the column alone.
struct Column {
  float scale, bias;
  int at;  // column of out
  bool live;
};

template <int KIND>
__device__ __forceinline__ Column column_of(const LinearView &p, int at) {
  Column c{1.0f, 0.0f, at, at < p.width};
  if (c.live) {
    if (KIND != kBf16) c.scale = p.ws[at];
    if (p.bias)
      c.bias = p.bias_f32 ? static_cast<const float *>(p.bias)[at]
                          : bf16_to_f32(static_cast<const uint16_t *>(p.bias)[at]);
  }
  return c;
}

// What U rows (`row`, `row` + `step`, .. below `end`) of a column need besides their sums.
template <int U>
struct Rows {
  float res[U], scale[U];
};

template <typename T, int U, bool FULL>
__device__ __forceinline__ void load_residual(const T *r, uint64_t by, int row, int step, int end, float (&res)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i, r += by)
    if (FULL || row + i * step < end) {
      if constexpr (sizeof(T) == 4) res[i] = *r;
      else res[i] = bf16_to_f32(*r);
    }
}

template <int KIND, int U>
__device__ __forceinline__ void load_rows(const LinearView &p, const Column &c, int row, int step, int end, Rows<U> &o) {
  const bool full = row + (U - 1) * step < end;
  if (p.res && c.live) {
    const uint64_t at = static_cast<uint64_t>(row) * p.res_stride + c.at, by = p.res_stride * static_cast<uint64_t>(step);
    if (p.res_f32) {
      const float *r = static_cast<const float *>(p.res) + at;
      if (full) load_residual<float, U, true>(r, by, row, step, end, o.res);
      else load_residual<float, U, false>(r, by, row, step, end, o.res);
    } else {
      const uint16_t *r = static_cast<const uint16_t *>(p.res) + at;
      if (full) load_residual<uint16_t, U, true>(r, by, row, step, end, o.res);
      else load_residual<uint16_t, U, false>(r, by, row, step, end, o.res);
    }
  }
  if constexpr (KIND != kBf16) {
    if (U % 4 == 0 && full && step == 1 && p.xs_vec) {  // row is a multiple of 16 here
#pragma unroll
      for (int i = 0; i < U / 4; ++i) {
        const float4 s = reinterpret_cast<const float4 *>(p.xs + row)[i];
        o.scale[4 * i] = s.x, o.scale[4 * i + 1] = s.y, o.scale[4 * i + 2] = s.z, o.scale[4 * i + 3] = s.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (row + i * step < end) o.scale[i] = p.xs[row + i * step];
    }
  }
}

// One row's 32 columns from `at` on into L2 (a row a lane).
__device__ __forceinline__ void prefetch_residual(const LinearView &p, int at, int row, int end) {
  const uint64_t size = p.res_f32 ? 4 : 2;
  if (at >= p.width) return;
  const uint64_t last = static_cast<uint64_t>(min(at + 31, p.width - 1) - at) * size;
  for (; row < end; row += 32) {
    const char *r = static_cast<const char *>(p.res) + (static_cast<uint64_t>(row) * p.res_stride + at) * size;
    asm volatile("prefetch.global.L2 [%0];\n prefetch.global.L2 [%1];\n" ::"l"(r), "l"(r + last));
  }
}

template <typename T, int U, bool FULL>
__device__ __forceinline__ void store_rows(T *o, uint64_t by, int row, int step, int end, const float (&v)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i, o += by)
    if (FULL || row + i * step < end) {
      if constexpr (sizeof(T) == 4) *o = v[i];
      else *o = f32_to_bf16(v[i]);
    }
}

// U rows of one column from their sums.
template <int KIND, int U>
__device__ __forceinline__ void finish(const LinearView &p, const Column &c, int row, int step, int end,
                                       const uint32_t (&raw)[U], const Rows<U> &in) {
  if (!c.live) return;
  float v[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if constexpr (KIND == kBf16) v[i] = __uint_as_float(raw[i]) + c.bias;
    else if constexpr (KIND == kInt8) v[i] = fmaf(static_cast<float>(static_cast<int32_t>(raw[i])) * in.scale[i], c.scale, c.bias);
    else v[i] = fmaf(__uint_as_float(raw[i]) * in.scale[i], c.scale, c.bias);
  }
  activate<U>(v, p.act, p.out_f32);
  if (p.res) {
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] += in.res[i];
  }
  const uint64_t at = static_cast<uint64_t>(row) * p.width + c.at, by = static_cast<uint64_t>(p.width) * step;
  const bool full = row + (U - 1) * step < end;
  if (p.out_f32) {
    float *o = static_cast<float *>(p.out) + at;
    if (full) store_rows<float, U, true>(o, by, row, step, end, v);
    else store_rows<float, U, false>(o, by, row, step, end, v);
  } else {
    uint16_t *o = static_cast<uint16_t *>(p.out) + at;
    if (full) store_rows<uint16_t, U, true>(o, by, row, step, end, v);
    else store_rows<uint16_t, U, false>(o, by, row, step, end, v);
  }
}

// Persistent CTAs (a cluster of `split` of them, which then has one item; or a
// pair) walk items of 128 weight rows (a pair 256) x up to NT rows of x.
//   warp 0     TMA producer over a ring of k-steps
//   warp 1     TMEM allocation, MMA issuer (one thread)
//   the others epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31, while the
//              next sums fill the other accumulator
// A split's CTAs sum a range of the k-steps each; the partial sums meet in
// shared memory and every CTA adds, in rank order, those of its share of rows.
// A pair's first CTA issues the MMAs of both (cta_group::2, M 256): each CTA
// brings its own weight rows and half the rows of x, both on the first one's
// barriers, and reads its own lanes' sums.  It halves the traffic of x into
// shared memory, which bounds large products: 48 KB a k-step come in at about 44
// bytes a clock (measured), against 512 clocks of bfloat16 MMAs, 256 of 8-bit
// ones.  (8192 x 4096 x 4096 int8: 117 us alone, 94 in pairs.)
// Every wait is bounded; a timeout sets kErrTimeout, marks the CTA dead (later
// waits return at once) and every role runs to the teardown.
template <int KIND, int NT, bool PAIR>
__global__ void __launch_bounds__(Shape<NT, PAIR>::kThreads, Shape<NT, PAIR>::kCtas)
    k_linear(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, LinearView p,
             uint32_t *err) {
  using S = Shape<NT, PAIR>;
  constexpr int kStep = KIND == kBf16 ? 64 : 128;  // elements of a k-step
  extern __shared__ __align__(128) uint8_t sm_raw[];
  uint8_t *sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(sm);
  auto bar = [&](int i) { return sbase + S::kBarOff + 8u * static_cast<uint32_t>(i); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + S::kBarOff + 8 * S::kBars);
  volatile uint32_t *dead = tmem_slot + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = PAIR ? 1 : p.split;
  const int rank = !PAIR && split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int half = PAIR ? static_cast<int>(cluster_rank()) : 0;  // of the pair
  const int first = PAIR ? blockIdx.x / 2 : blockIdx.x / split, step = PAIR ? gridDim.x / 2 : gridDim.x / split;
  const int k0 = static_cast<int>(static_cast<int64_t>(p.k_steps) * rank / split),
            k1 = static_cast<int>(static_cast<int64_t>(p.k_steps) * (rank + 1) / split);
  // an item's first weight row and row of x, of this CTA
  auto w_of = [&](int item) { return PAIR ? (item / p.x_tiles * 2 + half) * kLanes : item / p.x_tiles * kLanes; };
  auto x_of = [&](int item) { return item % p.x_tiles * p.tile; };
  if (tid == 0) {
    for (int i = 0; i < S::kBars; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar(i)), "r"(i >= S::kAccEmpty ? static_cast<uint32_t>(PAIR ? 2 * S::kEpi : S::kEpi) : 1u));
    *dead = 0u;
    mbar_init_fence();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                   "r"(S::kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                   "r"(S::kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // the other CTA's barriers and TMEM are there
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t st = 0, ph = 0, issued = 0;
      bool live = true;
      for (int item = first; item < p.items && live; item += step) {
        const int w0 = w_of(item), x0 = x_of(item) + half * (p.tile / 2);
        for (int k = k0; k < k1; ++k) {
          live = bounded_wait(bar(S::kEmpty + st), ph ^ 1u, dead, err);
          if (!live) break;
          const uint32_t base = sbase + st * S::kStage;
          if constexpr (PAIR) {
            // The first CTA's barrier counts both CTAs' bytes.  The other's may
            // land before they are announced: the arrival that announces them
            // is what the phase still waits for.
            if (half == 0) mbar_expect_tx_u32(bar(S::kFull + st), 2u * kBoxW + p.tile * 128u);
            const uint32_t full = in_rank(bar(S::kFull + st), 0);
            tma_box2d_pair(base, &wmap, k * kStep, w0, full);
            tma_box2d_pair(base + kBoxW, &xmap, k * kStep, x0, full);
          } else {
            mbar_expect_tx_u32(bar(S::kFull + st), kBoxW + p.tile * 128u);
            tma_box2d(base, &wmap, k * kStep, w0, bar(S::kFull + st));
            tma_box2d(base + kBoxW, &xmap, k * kStep, x0, bar(S::kFull + st));
          }
          ++issued;
          if (++st == S::kStages) st = 0, ph ^= 1u;
        }
      }
      // every box asked for has landed before the CTA may end (a pair's first CTA
      // waits for both, the other one for it at the last barrier)
      for (uint32_t i = half == 1 ? 0u : issued < S::kStages ? issued : S::kStages; i > 0; --i) {
        const uint32_t n = issued - i;
        for (uint32_t spins = 0; spins < kSpin && !mbar_try_wait_u32(bar(S::kFull + n % S::kStages), n / S::kStages & 1u); ++spins) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && half == 0) {
      const uint32_t id = idesc<KIND, PAIR>(p.tile);
      uint32_t st = 0, ph = 0;
      int n = 0;
      bool live = true;
      for (int item = first; item < p.items && live; item += step) {
        for (int from = k0; from < k1 && live; from += p.chunk, ++n) {
          live = bounded_wait(bar(S::kAccEmpty + (n & 1)), ((n >> 1) & 1) ^ 1u, dead, err);
          if (!live) break;
          tc_fence_after();
          const uint32_t d = tmem + (n & 1) * NT;
          const int to = min(k1, from + p.chunk);
          for (int k = from; k < to; ++k) {
            live = bounded_wait(bar(S::kFull + st), ph, dead, err);
            if (!live) break;
            tc_fence_after();
            const uint64_t a = sw128_desc(sbase + st * S::kStage), b = sw128_desc(sbase + st * S::kStage + kBoxW);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma<KIND, PAIR>(d, a + 2 * kk, b + 2 * kk, id, k != from || kk != 0);
            commit<PAIR>(bar(S::kEmpty + st));
            if (++st == S::kStages) st = 0, ph ^= 1u;
          }
          if (live) commit<PAIR>(bar(S::kAccFull + (n & 1)));
        }
      }
    }
  } else {
    constexpr int U = S::kRows;
    const int quarter = warp & 3, feat = 32 * quarter + lane, part = (warp - 2) / 4;
    // the tile's columns in 16s, dealt evenly to the warps of a quarter
    const int own = (p.tile / 16 + S::kEpi / 4 - 1) / (S::kEpi / 4) * 16, col0 = min(part * own, p.tile);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + col0;
    // this warp is done with an accumulator
    auto give_back = [&](int n) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) arrive_in_cluster(in_rank(bar(S::kAccEmpty + (n & 1)), 0));
        else mbar_arrive(bar(S::kAccEmpty + (n & 1)));
      }
    };
    int n = 0;
    bool live = true;
    for (int item = first; item < p.items && live; item += step) {
      const int w0 = w_of(item), x0 = x_of(item) + col0;
      const int cols = min(own, p.tile - col0), end = min(p.rows, x0 + cols);  // this warp's
      const Column c = column_of<KIND>(p, w0 + feat);
      // the residual into L2 and the first rows' residual and scales while the MMAs run
      Rows<U> ahead;
      if (split == 1 && x0 < end) {
        if (p.res) prefetch_residual(p, w0 + 32 * quarter, x0 + lane, end);
        load_rows<KIND, U>(p, c, x0, 1, end, ahead);
      }
      bool whole = true;  // the sums are whole as they lie in TMEM
      if constexpr (KIND != kInt8 && S::kSums) whole = k1 - k0 <= p.chunk;
      if (!whole) {
        // chunks are added in registers; their sum goes where the last one was
        constexpr int kWide = S::kCols < 32 || S::kEpi == 16 ? 16 : 32;
        float sum[S::kCols];
#pragma unroll
        for (int i = 0; i < S::kCols; ++i) sum[i] = 0.0f;
        for (int from = k0; from < k1; from += p.chunk, ++n) {
          live = bounded_wait(bar(S::kAccFull + (n & 1)), (n >> 1) & 1, dead, err);
          if (!live) break;
          __syncwarp();
          tc_fence_after();
          const uint32_t acc = lanes + (n & 1) * NT;
#pragma unroll
          for (int at = 0; at < S::kCols; at += kWide) {
            if (at >= cols) break;  // columns past the tile's end are read along, but not used
            uint32_t raw[kWide / 16][16];
#pragma unroll
            for (int j = 0; j < kWide / 16; ++j) tmem_ld16_nowait(acc + at + 16 * j, raw[j]);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < kWide; ++i) sum[at + i] = __fadd_rn(sum[at + i], __uint_as_float(raw[i / 16][i % 16]));
          }
          if (from + p.chunk >= k1) break;  // the last one's place is given back below
          give_back(n);
        }
        if (!live) break;
#pragma unroll
        for (int at = 0; at < S::kCols; at += 16)
          if (at < cols) tmem_st16(lanes + (n & 1) * NT + at, sum + at);
        tmem_wait_st();
      } else {
        live = bounded_wait(bar(S::kAccFull + (n & 1)), (n >> 1) & 1, dead, err);
        if (!live) break;
        __syncwarp();
        tc_fence_after();
      }
      const uint32_t acc = lanes + (n & 1) * NT;
      if (split > 1) {
#pragma unroll 1
        for (int at = 0; at < cols; at += 16) {
          uint32_t raw[16];
          tmem_ld16_nowait(acc + at, raw);
          tmem_wait_ld();
          uint32_t *part = reinterpret_cast<uint32_t *>(sm) + (col0 + at) * kLanes + feat;
#pragma unroll
          for (int i = 0; i < 16; ++i) part[i * kLanes] = raw[i];
        }
      } else {
#pragma unroll 1
        for (int at = x0; at < end; at += U) {
          uint32_t raw[U];
          const Rows<U> now = ahead;
          if constexpr (U == 16) tmem_ld16_nowait(acc + at - x0, raw);
          else tmem_ld8_nowait(acc + at - x0, raw);
          if (at + U < end) load_rows<KIND, U>(p, c, at + U, 1, end, ahead);
          tmem_wait_ld();
          finish<KIND, U>(p, c, at, 1, end, raw, now);
        }
      }
      give_back(n);
      ++n;
    }
  }
  __syncwarp();
  if (split > 1) {
    cluster_barrier();
    if (warp >= 2) {
      constexpr int U = NT <= 32 ? 2 : NT <= 64 ? 4 : 8, R = NT <= 32 ? 8 : 4;  // rows and ranks whose sums a thread asks for at once
      const int w0 = w_of(first), x0 = x_of(first);
      const int feat = 32 * (warp & 3) + lane, end = min(p.tile, p.rows - x0);
      const int step1 = split * (S::kEpi / 4);  // rows dealt to ranks, then to the warps of a quarter
      const Column c = column_of<KIND>(p, w0 + feat);
      for (int row = rank + (warp - 2) / 4 * split; row < end; row += U * step1) {
        uint32_t raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i) raw[i] = 0u;
        Rows<U> in;
        load_rows<KIND, U>(p, c, x0 + row, step1, x0 + end, in);
        for (int r0 = 0; r0 < split; r0 += R) {
          uint32_t part[R][U];
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < U; ++i)
              part[r][i] = r0 + r < split && row + i * step1 < end
                               ? peer_word(sbase + 4u * static_cast<uint32_t>((row + i * step1) * kLanes + feat), r0 + r)
                               : 0u;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < U; ++i)
              raw[i] = KIND == kInt8 ? raw[i] + part[r][i]
                                     : __float_as_uint(__fadd_rn(__uint_as_float(raw[i]), __uint_as_float(part[r][i])));
        }
        finish<KIND, U>(p, c, x0 + row, step1, x0 + end, raw, in);
      }
    }
    __syncwarp();
    cluster_barrier();  // no CTA ends while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // neither CTA's memory goes while the other's MMAs, copies or arrivals may reach it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kTmemCols));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kTmemCols));
  }
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no -lcuda).
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn linear_encode_fn() {
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

// [rows][width] as boxes of 128 bytes x box_rows, 128-byte swizzle, zero past the ends.
bool make_map(CUtensorMap *map, const void *base, bool bf16, uint64_t rows, uint64_t width, uint64_t stride_bytes,
              int box_rows) {
  EncodeTiledFn fn = linear_encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {width, rows};
  const cuuint64_t strides[1] = {stride_bytes};
  const cuuint32_t box[2] = {bf16 ? 64u : 128u, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base),
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            // a k-step takes 128 bytes of many rows; DRAM gives the next k-step's along (97 -> 88 us for a head)
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, int NT, bool PAIR = false>
cudaError_t launch(const CUtensorMap &wm, const CUtensorMap &xm, LinearView p, int sms, cudaStream_t s) {
  using S = Shape<NT, PAIR>;
  cudaError_t e = cudaFuncSetAttribute(k_linear<KIND, NT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const int slots = sms * S::kCtas;
  // Few tiles leave SMs without work: a cluster of CTAs then shares an item's
  // k-steps, at least four each so that the ring fills.
  p.split = 1;
  while (!PAIR && p.split < 8 && p.items * p.split * 2 <= slots && p.k_steps / (p.split * 2) >= 4 && p.items * p.split < sms)
    p.split *= 2;
  // The tensor core drops what it shifts out of its float32 sums, a bias of
  // about 2^-25 an addition that grows with their number (measured: 2.2e-6 of
  // the result after 128 of them).  Results that stay float32 are summed 16
  // additions at a time (32 in pairs, whose epilogue is busier) and those sums
  // added with rounding; bfloat16 results keep the bias (2^-12 at the largest width,
  // where their rounding takes up to 2^-8), int8 sums are exact.
  p.chunk = KIND != kInt8 && p.out_f32 ? (PAIR ? 8 : 4) : p.k_steps;
  const int cluster = PAIR ? 2 : p.split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.split > 1 ? p.items * p.split : std::min(p.items, slots / cluster) * cluster));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, k_linear<KIND, NT, PAIR>, wm, xm, p, device_error_word());
}

bool misaligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <int KIND>
int run(const FnLinearArgs *a, LinearView &p, cudaStream_t s, std::string &err) {
  constexpr uint64_t size = KIND == kBf16 ? 2 : 1;
  const int sms = device_info().sms;
  const bool sums = KIND != kInt8 && p.out_f32;
  // Pairs from 257 rows on, where there are two tiles of weight rows.  x 2048 > 5120,
  // one CTA alone and in pairs, us: float32 results 26 and 18 at 512 rows, 60 and 44
  // at 2,000, 129 and 114 at 5,000 (but 15.5 and 16.9 at 384); bfloat16 80 and 79 at
  // 5,000, 37 and 38 at 2,000, 14.7 and 15.9 at 512; int8 (e4m3 much the same) 46.5
  // and 46.5 at 5,000, 23 and 24.5 at 2,000, 10.5 and 11.5 at 512; 8192 x 4096 x 4096
  // int8 117 and 94.
  const bool pair = p.rows > 256 && p.width > kLanes;
  const int nt = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : p.rows <= 128 ? 128 : !sums ? 256 : pair ? 192 : 128;
  const int64_t lanes = pair ? 2 * kLanes : kLanes, w_tiles = (p.width + lanes - 1) / lanes, step = pair ? 32 : 16;
  p.tile = static_cast<int>(std::min<int64_t>(nt, (p.rows + step - 1) / step * step));
  if (p.rows > nt) {
    // Tiles as wide as leaves the last round of items no emptier than the
    // others: fewest rounds x columns (and 48 columns' time for an item's start
    // and end).  1024 x 5120: 7 tiles of 160 in two rounds, not 4 of 256 in two.
    // (5000 x 2048 > 5120 bfloat16: 118 us without the 48, 104 with 16, 79.5 with 48,
    // 79.3 with 128; e4m3 70, 61, 49, 49; from 600 to 3,000 rows all alike.)
    const int64_t tiles0 = (p.rows + nt - 1) / nt, slots = pair ? sms / 2 : sms;
    int64_t least = INT64_MAX;
    for (int64_t n = tiles0; n <= 2 * tiles0 && n < tiles0 + 64; ++n) {
      const int64_t wide = ((p.rows + n - 1) / n + step - 1) / step * step;
      const int64_t time = (w_tiles * ((p.rows + wide - 1) / wide) + slots - 1) / slots * (wide + 48);
      if (time < least) least = time, p.tile = static_cast<int>(wide);
    }
  }
  p.k_steps = static_cast<int>((a->in_width * size + 127) / 128);
  p.x_tiles = (p.rows + p.tile - 1) / p.tile;
  const int64_t items = w_tiles * p.x_tiles;
  if (items > 0x1FFFFFFF) { err = "too many rows for one call"; return FNMOE_ERR_SHAPE; }
  p.items = static_cast<int>(items);
  // a single row's stride is not used, but has to be a valid one
  const uint64_t row = (a->in_width * size + 15) / 16 * 16;
  CUtensorMap wm, xm;
  if (!make_map(&wm, a->weight, KIND == kBf16, a->out_width, a->in_width, a->out_width > 1 ? a->weight_stride * size : row, kLanes) ||
      !make_map(&xm, a->x, KIND == kBf16, a->rows, a->in_width, a->rows > 1 ? a->x_stride * size : row, pair ? p.tile / 2 : p.tile)) {
    err = "linear: no tensor map for x or weight";
    return FNMOE_ERR_LAUNCH;
  }
  cudaError_t e;
  switch (nt) {
    case 16: e = launch<KIND, 16>(wm, xm, p, sms, s); break;
    case 32: e = launch<KIND, 32>(wm, xm, p, sms, s); break;
    case 64: e = launch<KIND, 64>(wm, xm, p, sms, s); break;
    case 128: e = launch<KIND, 128>(wm, xm, p, sms, s); break;
    case 192:
      if constexpr (KIND != kInt8) e = launch<KIND, 192, true>(wm, xm, p, sms, s);
      else e = cudaErrorInvalidValue;
      break;
    default: e = pair ? launch<KIND, 256, true>(wm, xm, p, sms, s) : launch<KIND, 256>(wm, xm, p, sms, s); break;
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return FNMOE_OK;
  err = std::string("linear: ") + cudaGetErrorString(e);
  return FNMOE_ERR_LAUNCH;
}

}  // namespace

int linear(const FnLinearArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (a->type > FNMOE_LINEAR_E4M3 || a->activation > FNMOE_ACT_RELU) {
    err = "unknown type or activation";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (a->bias_dtype > FNMOE_DTYPE_F32 || a->residual_dtype > FNMOE_DTYPE_F32 || a->out_dtype > FNMOE_DTYPE_F32) {
    err = "bias, residual and out must be bfloat16 or float32";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (a->in_width == 0 || a->out_width == 0 || a->in_width > kMaxWidth || a->out_width > 0x7FFFFF00u || a->rows > 0x7FFFFF00u) {
    err = "in_width must be between 1 and " + std::to_string(kMaxWidth) + ", out_width positive, both and rows below 2^31 - 256";
    return FNMOE_ERR_SHAPE;
  }
  if (a->rows == 0) return FNMOE_OK;
  if (!a->x || !a->weight || !a->out) { err = "x, weight and out are required"; return FNMOE_ERR_NULL; }
  const bool q8 = a->type != FNMOE_LINEAR_BF16;
  if (q8 != (a->x_scale != nullptr) || q8 != (a->weight_scale != nullptr)) {
    err = "8-bit x and weight need x_scale and weight_scale, bfloat16 ones have none";
    return FNMOE_ERR_NULL;
  }
  const uint64_t size = q8 ? 1 : 2;
  if ((a->rows > 1 && a->x_stride < a->in_width) || (a->out_width > 1 && a->weight_stride < a->in_width) ||
      (a->residual && a->rows > 1 && a->residual_stride < a->out_width)) {
    err = "row strides must cover a row";
    return FNMOE_ERR_SHAPE;
  }
  if (misaligned(a->x, 16) || misaligned(a->weight, 16) || (a->rows > 1 && a->x_stride * size % 16) ||
      (a->out_width > 1 && a->weight_stride * size % 16)) {
    err = "x and weight must start on 16-byte boundaries and have row strides that are multiples of 16 bytes";
    return FNMOE_ERR_VALUE;
  }
  auto bytes = [](uint32_t d) { return d == FNMOE_DTYPE_F32 ? uintptr_t(4) : uintptr_t(2); };
  if (misaligned(a->x_scale, 4) || misaligned(a->weight_scale, 4) || misaligned(a->bias, bytes(a->bias_dtype)) ||
      misaligned(a->residual, bytes(a->residual_dtype)) || misaligned(a->out, bytes(a->out_dtype))) {
    err = "arrays must be aligned to their elements";
    return FNMOE_ERR_VALUE;
  }
  const uint64_t rows = a->rows, width = a->out_width, rs = bytes(a->residual_dtype), os = bytes(a->out_dtype);
  const Span out{a->out, rows * width * os};
  const bool in_place = a->out == a->residual && a->out_dtype == a->residual_dtype && (rows == 1 || a->residual_stride == width);
  if (out.meets(Span{a->x, ((rows - 1) * a->x_stride + a->in_width) * size}) ||
      out.meets(Span{a->weight, ((width - 1) * a->weight_stride + a->in_width) * size}) ||
      out.meets(Span{a->x_scale, rows * 4}) || out.meets(Span{a->weight_scale, width * 4}) ||
      out.meets(Span{a->bias, width * bytes(a->bias_dtype)}) ||
      (!in_place && out.meets(Span{a->residual, ((rows - 1) * a->residual_stride + width) * rs}))) {
    err = "out overlaps an input (it may be residual where types and strides are the same)";
    return FNMOE_ERR_VALUE;
  }
  LinearView p{};
  p.xs = a->x_scale;
  p.ws = a->weight_scale;
  p.bias = a->bias;
  p.res = a->residual;
  p.out = a->out;
  p.res_stride = a->residual_stride;
  p.rows = static_cast<int>(a->rows);
  p.width = static_cast<int>(a->out_width);
  p.act = a->activation;
  p.bias_f32 = a->bias_dtype == FNMOE_DTYPE_F32;
  p.res_f32 = a->residual_dtype == FNMOE_DTYPE_F32;
  p.out_f32 = a->out_dtype == FNMOE_DTYPE_F32;
  p.xs_vec = !misaligned(a->x_scale, 16);
  switch (a->type) {
    case FNMOE_LINEAR_INT8: return run<kInt8>(a, p, s, err);
    case FNMOE_LINEAR_E4M3: return run<kE4m3>(a, p, s, err);
    default: return run<kBf16>(a, p, s, err);
  }
}

}  // namespace fnmoe
