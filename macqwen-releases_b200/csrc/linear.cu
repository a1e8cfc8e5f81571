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
// to 131072 keep 127^2 K below 2^31).  The epilogue works on float32 and rounds
// once, to the output's type.
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
constexpr int kThreads = 192;
constexpr uint32_t kMaxWidth = 131072;

enum Kind { kBf16 = FNMOE_LINEAR_BF16, kInt8 = FNMOE_LINEAR_INT8, kE4m3 = FNMOE_LINEAR_E4M3 };

struct LinearView {
  const float *xs, *ws;
  const void *bias, *res;
  void *out;
  uint64_t res_stride;
  int rows, width, k_steps;  // rows of x, columns of out, k-steps of 128 bytes
  int x_tiles, items;
  int split;                 // CTAs of a cluster that share an item's k-steps
  uint32_t act;
  bool bias_f32, res_f32, out_f32;
};

template <int NT>
struct Shape {
  static constexpr int kBoxX = NT * 128;
  static constexpr int kStage = kBoxW + kBoxX;
  // small tiles leave room for a second CTA on the SM
  static constexpr int kStages = NT <= 32 ? 5 : NT <= 64 ? 4 : NT <= 128 ? 6 : 4;
  static constexpr int kCtas = NT <= 64 ? 2 : 1;
  static constexpr int kBarOff = kStages * kStage;
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + 2,
                       kBars = kAccEmpty + 2;
  static constexpr int kSmem = kBarOff + 8 * kBars + 16 + 1024;  // + TMEM slot, dead flag, 1 KiB alignment
  static constexpr uint32_t kTmemCols = 2 * NT < 32 ? 32 : 2 * NT;
  static_assert(kCtas * (kSmem + 1024) <= 227 * 1024, "shared memory");
  static_assert(NT * kLanes * 4 <= kBarOff, "a split's partial sums lie in the ring");
};

// Instruction descriptor: D float32 (s32 for int8), both operands K-major,
// N = NT, M = 128; operand formats bf16, signed 8-bit or e4m3.
template <int KIND, int NT>
constexpr uint32_t idesc() {
  const uint32_t d = KIND == kInt8 ? 2u : 1u, ab = KIND == kE4m3 ? 0u : 1u;
  return (d << 4) | (ab << 7) | (ab << 10) | (static_cast<uint32_t>(NT >> 3) << 17) |
         (static_cast<uint32_t>(kLanes >> 4) << 24);
}

template <int KIND, int NT>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  constexpr uint32_t id = idesc<KIND, NT>();
  if constexpr (KIND == kBf16)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
  else if constexpr (KIND == kInt8)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
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

// exp and erfc by CUDA's functions where the result stays float32; where it is
// rounded to bfloat16 (2^-9) the approximate exponential and quotient (2^-21)
// cost nothing that shows and keep the epilogue shorter than a tile's MMAs.
__device__ __forceinline__ float activate(float a, uint32_t act, bool f32) {
  switch (act) {
    case FNMOE_ACT_SILU:
      return f32 ? __fdiv_rn(a, 1.0f + expf(-a)) : __fdividef(a, 1.0f + __expf(-a));
    case FNMOE_ACT_GELU: return 0.5f * a * erfcf(-0.70710678118654752f * a);
    case FNMOE_ACT_RELU: return a < 0.0f ? 0.0f : a;
    default: return a;
  }
}

// This lane's part of out's row: everything that depends on the column alone.
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

// U rows of one column from raw accumulators: the residual's loads go out together.
template <int KIND, int U>
__device__ __forceinline__ void finish(const LinearView &p, const Column &c, int row, const uint32_t (&raw)[U]) {
  if (!c.live) return;
  float res[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    res[i] = 0.0f;
    if (p.res && row + i < p.rows) {
      const uint64_t at = static_cast<uint64_t>(row + i) * p.res_stride + c.at;
      res[i] = p.res_f32 ? static_cast<const float *>(p.res)[at] : bf16_to_f32(static_cast<const uint16_t *>(p.res)[at]);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (row + i >= p.rows) break;
    float v = KIND == kInt8 ? static_cast<float>(static_cast<int32_t>(raw[i])) : __uint_as_float(raw[i]);
    if (KIND != kBf16) v = v * p.xs[row + i] * c.scale;
    v = activate(v + c.bias, p.act, p.out_f32) + res[i];
    const uint64_t at = static_cast<uint64_t>(row + i) * p.width + c.at;
    if (p.out_f32) static_cast<float *>(p.out)[at] = v;
    else static_cast<uint16_t *>(p.out)[at] = f32_to_bf16(v);
  }
}

// Persistent CTAs (a cluster of `split` of them, which then has one item)
// walk items of 128 weight rows x NT rows of x.
//   warp 0     TMA producer over a ring of k-steps
//   warp 1     TMEM allocation, MMA issuer (one thread)
//   warps 2-5  epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31, while the
//              next item's MMAs fill the other accumulator
// A split's CTAs sum a range of the k-steps each; the partial sums meet in
// shared memory and every CTA adds, in rank order, those of its share of rows.
// Every wait is bounded; a timeout sets kErrTimeout, marks the CTA dead (later
// waits return at once) and every role runs to the teardown.
template <int KIND, int NT>
__global__ void __launch_bounds__(kThreads, Shape<NT>::kCtas) k_linear(const __grid_constant__ CUtensorMap wmap,
                                                                       const __grid_constant__ CUtensorMap xmap,
                                                                       LinearView p, uint32_t *err) {
  using S = Shape<NT>;
  constexpr int kStep = KIND == kBf16 ? 64 : 128;  // elements of a k-step
  extern __shared__ __align__(128) uint8_t sm_raw[];
  uint8_t *sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(sm);
  auto bar = [&](int i) { return sbase + S::kBarOff + 8u * static_cast<uint32_t>(i); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + S::kBarOff + 8 * S::kBars);
  volatile uint32_t *dead = tmem_slot + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int first = blockIdx.x / p.split, step = gridDim.x / p.split;
  const int k0 = static_cast<int>(static_cast<int64_t>(p.k_steps) * rank / p.split),
            k1 = static_cast<int>(static_cast<int64_t>(p.k_steps) * (rank + 1) / p.split);
  if (tid == 0) {
    for (int i = 0; i < S::kBars; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar(i)), "r"(i >= S::kAccEmpty ? 4u : 1u));
    *dead = 0u;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(S::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t st = 0, ph = 0, issued = 0;
      bool live = true;
      for (int item = first; item < p.items && live; item += step) {
        const int w0 = item / p.x_tiles * kLanes, x0 = item % p.x_tiles * NT;
        for (int k = k0; k < k1; ++k) {
          live = bounded_wait(bar(S::kEmpty + st), ph ^ 1u, dead, err);
          if (!live) break;
          mbar_expect_tx_u32(bar(S::kFull + st), S::kStage);
          const uint32_t base = sbase + st * S::kStage;
          tma_box2d(base, &wmap, k * kStep, w0, bar(S::kFull + st));
          tma_box2d(base + kBoxW, &xmap, k * kStep, x0, bar(S::kFull + st));
          ++issued;
          if (++st == S::kStages) st = 0, ph ^= 1u;
        }
      }
      // every box asked for has landed before the CTA may end
      for (uint32_t i = issued < S::kStages ? issued : S::kStages; i > 0; --i) {
        const uint32_t n = issued - i;
        for (uint32_t spins = 0; spins < kSpin && !mbar_try_wait_u32(bar(S::kFull + n % S::kStages), n / S::kStages & 1u); ++spins) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t st = 0, ph = 0;
      int n = 0;
      bool live = true;
      for (int item = first; item < p.items && live; item += step, ++n) {
        live = bounded_wait(bar(S::kAccEmpty + (n & 1)), ((n >> 1) & 1) ^ 1u, dead, err);
        if (!live) break;
        tc_fence_after();
        const uint32_t d = tmem + (n & 1) * NT;
        for (int k = k0; k < k1; ++k) {
          live = bounded_wait(bar(S::kFull + st), ph, dead, err);
          if (!live) break;
          tc_fence_after();
          const uint64_t a = sw128_desc(sbase + st * S::kStage), b = sw128_desc(sbase + st * S::kStage + kBoxW);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma<KIND, NT>(d, a + 2 * kk, b + 2 * kk, k != k0 || kk != 0);
          umma_commit(bar(S::kEmpty + st));
          if (++st == S::kStages) st = 0, ph ^= 1u;
        }
        if (live) umma_commit(bar(S::kAccFull + (n & 1)));
      }
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    int n = 0;
    for (int item = first; item < p.items; item += step, ++n) {
      if (!bounded_wait(bar(S::kAccFull + (n & 1)), (n >> 1) & 1, dead, err)) break;
      __syncwarp();
      tc_fence_after();
      const int w0 = item / p.x_tiles * kLanes, x0 = item % p.x_tiles * NT;
      const int feat = 32 * quarter + lane;
      const uint32_t acc = lanes + (n & 1) * NT;
      const Column c = column_of<KIND>(p, w0 + feat);
#pragma unroll 1
      for (int at = 0; at < NT; at += 16) {
        uint32_t raw[16];
        tmem_ld16_nowait(acc + at, raw);
        tmem_wait_ld();
        if (p.split > 1) {
          uint32_t *part = reinterpret_cast<uint32_t *>(sm) + at * kLanes + feat;
#pragma unroll
          for (int i = 0; i < 16; ++i) part[i * kLanes] = raw[i];
        } else {
          finish<KIND, 16>(p, c, x0 + at, raw);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S::kAccEmpty + (n & 1)));
    }
  }
  __syncwarp();
  if (p.split > 1) {
    cluster_barrier();
    if (warp >= 2) {
      const int w0 = first / p.x_tiles * kLanes, x0 = first % p.x_tiles * NT;
      const int feat = 32 * (warp & 3) + lane;
      const Column c = column_of<KIND>(p, w0 + feat);
      for (int row = rank; row < NT && x0 + row < p.rows; row += p.split) {
        const uint32_t a = sbase + 4u * static_cast<uint32_t>(row * kLanes + feat);
        uint32_t part[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) part[r] = r < p.split ? peer_word(a, r) : 0u;
        uint32_t raw[1];
        if (KIND == kInt8) {
          raw[0] = 0u;
#pragma unroll
          for (int r = 0; r < 8; ++r) raw[0] += part[r];
        } else {
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 8; ++r) sum = __fadd_rn(sum, __uint_as_float(part[r]));
          raw[0] = __float_as_uint(sum);
        }
        finish<KIND, 1>(p, c, x0 + row, raw);
      }
    }
    __syncwarp();
    cluster_barrier();  // no CTA ends while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kTmemCols));
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
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, int NT>
cudaError_t launch(const CUtensorMap &wm, const CUtensorMap &xm, LinearView p, int sms, cudaStream_t s) {
  using S = Shape<NT>;
  cudaError_t e = cudaFuncSetAttribute(k_linear<KIND, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const int slots = sms * S::kCtas;
  // Few tiles leave SMs without work: a cluster of CTAs then shares an item's
  // k-steps, at least four each so that the ring fills.
  p.split = 1;
  while (p.split < 8 && p.items * p.split * 2 <= slots && p.k_steps / (p.split * 2) >= 4 && p.items * p.split < sms)
    p.split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.split > 1 ? p.items * p.split : std::min(p.items, slots)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.split > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.split);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, k_linear<KIND, NT>, wm, xm, p, device_error_word());
}

bool misaligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

template <int KIND>
int run(const FnLinearArgs *a, LinearView &p, cudaStream_t s, std::string &err) {
  constexpr uint64_t size = KIND == kBf16 ? 2 : 1;
  const int nt = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : p.rows <= 128 ? 128 : 256;
  p.k_steps = static_cast<int>((a->in_width * size + 127) / 128);
  p.x_tiles = (p.rows + nt - 1) / nt;
  const int64_t items = static_cast<int64_t>((p.width + static_cast<int64_t>(kLanes) - 1) / kLanes) * p.x_tiles;
  if (items > 0x1FFFFFFF) { err = "too many rows for one call"; return FNMOE_ERR_SHAPE; }
  p.items = static_cast<int>(items);
  // a single row's stride is not used, but has to be a valid one
  const uint64_t row = (a->in_width * size + 15) / 16 * 16;
  CUtensorMap wm, xm;
  if (!make_map(&wm, a->weight, KIND == kBf16, a->out_width, a->in_width, a->out_width > 1 ? a->weight_stride * size : row, kLanes) ||
      !make_map(&xm, a->x, KIND == kBf16, a->rows, a->in_width, a->rows > 1 ? a->x_stride * size : row, nt)) {
    err = "linear: no tensor map for x or weight";
    return FNMOE_ERR_LAUNCH;
  }
  const int sms = device_info().sms;
  cudaError_t e;
  switch (nt) {
    case 16: e = launch<KIND, 16>(wm, xm, p, sms, s); break;
    case 32: e = launch<KIND, 32>(wm, xm, p, sms, s); break;
    case 64: e = launch<KIND, 64>(wm, xm, p, sms, s); break;
    case 128: e = launch<KIND, 128>(wm, xm, p, sms, s); break;
    default: e = launch<KIND, 256>(wm, xm, p, sms, s); break;
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
  switch (a->type) {
    case FNMOE_LINEAR_INT8: return run<kInt8>(a, p, s, err);
    case FNMOE_LINEAR_E4M3: return run<kE4m3>(a, p, s, err);
    default: return run<kBf16>(a, p, s, err);
  }
}

}  // namespace fnmoe
