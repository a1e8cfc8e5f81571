// sample.cu -- one token a row of logits by temperature, top-k, top-p and min-p
// from a given uniform number, in one launch that reads the logits once.
//
// Ranked by falling logit, equal ones by rising index, each filter keeps a
// prefix, so together they keep the tokens up to one place: a (logit, index)
// pair, found by counting instead of sorting.  The row lies in the shared
// memory of a cluster's CTAs; a histogram of the logits (1024 equal ranges)
// names the range in which the place falls, the few tokens of that range are
// gathered and ranked against one another.  A range that holds too many of
// them (ties, outliers) is divided again, by the bits of (logit, index), until
// it does not.  The draw then walks the kept tokens by index.
//
// Weights are exp((l - max) / T) in float64, held as integers of 2^-44 of the
// largest: sums are then exact and do not depend on the order of threads or
// atomics, and a vocabulary of 2^18 stays below 2^62.  Float32 weights (2^-24)
// would draw another token than the definition once in some thousand rows of a
// flat distribution, whose borders lie 2^-17 apart.
#include <cuda_bf16.h>
#include <stdint.h>

#include <algorithm>

#include "async.cuh"
#include "common.cuh"
#include "dense.cuh"
#include "moe_kernels.cuh"

namespace fnmoe {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kList = 1024;       // tokens that are ranked against one another
constexpr int kIndexBits = 18;    // FNMOE_SAMPLE_MAX_VOCAB
constexpr int kPlaceBits = 32 + kIndexBits;
constexpr uint64_t kAll = ~0ull;  // a place past every token
constexpr double kOne = 0x1p44;   // the largest weight
constexpr float kMinusInf = -__builtin_inff();

struct SampleView {
  const void *logits;
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int32_t *top_ks;
  int64_t *tokens;
  float *logprobs;
  uint64_t stride;
  int vocab, slice;  // tokens of a row, and of a CTA's part of it
  int ctas;          // of a cluster
  float temperature, top_p, min_p;
  int32_t top_k;
};

// What the CTAs of a cluster tell one another, each in its own copy.
struct Shared {
  uint32_t count[kBins];                        // this CTA's histogram
  uint32_t mass_lo[kBins], mass_hi[kBins];      // and its weights
  uint64_t list_at[kList], list_w[kList];       // (rank 0) gathered tokens: places and weights
  uint64_t warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  float warp_max[kWarps], warp_min[kWarps];
  float row_max, row_min;                       // of this CTA's part
  uint64_t part_mass;                           // of this CTA's bins, or of its kept tokens
  uint32_t part_count;
  uint32_t list_n;                              // (rank 0)
  uint32_t best;                                // this CTA's lowest index of the largest logit
  // the range in which the place falls (written to every copy by the CTA that finds it)
  uint32_t hit_bin, hit_count, hit_before_count;
  uint64_t hit_mass, hit_before_mass;
  uint64_t place;                               // the last kept token (written to every copy by rank 0)
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The address in the cluster's CTA `rank` of what lies at `p` here, as a generic pointer.
template <typename T>
__device__ __forceinline__ T *at_rank(T *p, uint32_t rank) {
  uint64_t out;
  asm volatile("mapa.u64 %0, %1, %2;\n" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<T *>(out);
}

template <typename T>
__device__ __forceinline__ float logit(const T *p);
template <>
__device__ __forceinline__ float logit<uint16_t>(const uint16_t *p) { return bf16_to_f32(*p); }
template <>
__device__ __forceinline__ float logit<float>(const float *p) { return *p; }

// Larger logits first, then lower indices; -0 counts as 0.
__device__ __forceinline__ uint64_t place_of(float l, uint32_t index) {
  const uint32_t b = __float_as_uint(__fadd_rn(l, 0.0f));
  const uint32_t up = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(~up) << kIndexBits) | index;
}

// A row's weights.
struct Weights {
  float top;
  double inv_t;
  __device__ __forceinline__ double exponent(float l) const {
    return l == top ? 0.0 : (static_cast<double>(l) - static_cast<double>(top)) * inv_t;
  }
  static __device__ __forceinline__ uint64_t of(double x) {
    return x > -32.0 ? static_cast<uint64_t>(__double2ll_rn(exp(x) * kOne)) : 0ull;
  }
};

// Exclusive prefix over the CTA's threads of (count, mass), and their totals.
__device__ __forceinline__ void scan(uint32_t &count, uint64_t &mass, uint32_t &total_count, uint64_t &total_mass,
                                     Shared &s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t c = count;
  uint64_t m = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t pc = __shfl_up_sync(0xFFFFFFFFu, c, o);
    const uint64_t pm = __shfl_up_sync(0xFFFFFFFFu, m, o);
    if (lane >= o) c += pc, m += pm;
  }
  __syncthreads();
  if (lane == 31) s.warp_count[warp] = c, s.warp_sum[warp] = m;
  __syncthreads();
  uint32_t before_c = 0;
  uint64_t before_m = 0;
  total_count = 0;
  total_mass = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i == warp) before_c = total_count, before_m = total_mass;
    total_count += s.warp_count[i];
    total_mass += s.warp_sum[i];
  }
  count = before_c + c - count;
  mass = before_m + m - mass;
}

// One row, in a cluster of p.ctas CTAs.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(SampleView p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.ctas;
  const uint32_t rank = blockIdx.x % p.ctas;
  const uint32_t begin = rank * static_cast<uint32_t>(p.slice);
  const int n = max(0, min(p.slice, p.vocab - static_cast<int>(begin)));
  pdl_wait();
  pdl_trigger();

  // ---- the CTA's part of the row into shared memory, with its largest and least logit ----
  constexpr int kVec = 16 / sizeof(T);
  const T *src = static_cast<const T *>(p.logits) + static_cast<uint64_t>(row) * p.stride + begin;
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  T *data = reinterpret_cast<T *>(smem + (sizeof(Shared) + 15) / 16 * 16) + skew;  // aligned like src
  float hi = kMinusInf, lo = -kMinusInf;
  auto meet = [&](float l) {  // NaN leaves both alone
    hi = fmaxf(hi, l);
    if (l > kMinusInf) lo = fminf(lo, l);
  };
  const int head = min(n, (kVec - skew) % kVec), vecs = (n - head) / kVec;
  for (int i = tid; i < head; i += kThreads) {
    data[i] = src[i];
    meet(logit<T>(src + i));
  }
  const uint4 *src4 = reinterpret_cast<const uint4 *>(src + head);
  uint4 *data4 = reinterpret_cast<uint4 *>(data + head);
  auto take = [&](uint4 v, int i) {
    data4[i] = v;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        meet(__uint_as_float(w[e]));
      } else {
        meet(__uint_as_float(w[e] << 16));
        meet(__uint_as_float(w[e] & 0xFFFF0000u));
      }
    }
  };
  int v0 = tid;
  for (; v0 + 3 * kThreads < vecs; v0 += 4 * kThreads) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = src4[v0 + j * kThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j) take(v[j], v0 + j * kThreads);
  }
  for (; v0 < vecs; v0 += kThreads) take(src4[v0], v0);
  for (int i = head + vecs * kVec + tid; i < n; i += kThreads) {
    data[i] = src[i];
    meet(logit<T>(src + i));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
  }
  if (lane == 0) s.warp_max[warp] = hi, s.warp_min[warp] = lo;
  if (tid == 0) s.list_n = 0u, s.best = 0xFFFFFFFFu;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kWarps; ++i) hi = fmaxf(hi, s.warp_max[i]), lo = fminf(lo, s.warp_min[i]);
    s.row_max = hi;
    s.row_min = lo;
  }
  cluster_barrier();
  hi = kMinusInf, lo = -kMinusInf;
  for (int r = 0; r < p.ctas; ++r) {
    hi = fmaxf(hi, at_rank(&s, r)->row_max);
    lo = fminf(lo, at_rank(&s, r)->row_min);
  }

  // ---- the row's settings ----
  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  const Weights weights{hi, 1.0 / static_cast<double>(t)};
  // the largest logit: asked for, or all that there is
  if (!(t > 0.0f) || top_k == 1 || !(top_p > 0.0f) || !(hi > kMinusInf)) {
    uint32_t best = 0xFFFFFFFFu;
    if (hi > kMinusInf)
      for (int i = tid; i < n; i += kThreads)
        if (logit<T>(data + i) == hi) {
          best = begin + static_cast<uint32_t>(i);
          break;
        }
    best = __reduce_min_sync(0xFFFFFFFFu, best);
    if (lane == 0 && best != 0xFFFFFFFFu) atomicMin(&s.best, best);
    cluster_barrier();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < p.ctas; ++r) best = min(best, at_rank(&s, r)->best);
      p.tokens[row] = best == 0xFFFFFFFFu ? -1 : static_cast<int64_t>(best);
      if (p.logprobs) p.logprobs[row] = 0.0f;
    }
    cluster_barrier();
    return;
  }

  // ---- the place of the last kept token ----
  uint64_t place = kAll;
  // Tokens up to `place` (so far): the first `want_count` of them, or (by_mass)
  // those before whose place less than `share` of their weights lies.
  auto narrow = [&](const bool by_mass, const uint32_t want_count, const double share) {
    // ranges of the first round: equal parts of the logits that can matter
    float span = __fsub_rn(hi, lo);
    if (by_mass) span = fminf(span, 32.0f * t);
    const float per = span > 0.0f ? __fdiv_rn(static_cast<float>(kBins), span) : 0.0f;
    auto range_of = [&](float l) {  // rises (weakly) with falling logits
      const int b = static_cast<int>(__fmul_rn(__fsub_rn(hi, l), per));
      return static_cast<uint32_t>(min(max(b, 0), kBins - 1));
    };
    uint32_t range = 0;     // chosen in the first round
    uint64_t prefix = 0;    // of the place, chosen in later rounds
    uint32_t before_count = 0;
    uint64_t before_mass = 0, target = 0;
    for (int round = 0;; ++round) {
      const int shift = kPlaceBits - 10 * round;  // of the later rounds' digits: 40, 30, .., 0
      auto member = [&](float l, uint64_t at) {
        if (!(l > kMinusInf) || at > place) return false;
        if (round == 0) return true;
        return range_of(l) == range && (round == 1 || (at >> (shift + 10)) == prefix);
      };
      auto bin_of = [&](float l, uint64_t at) {
        return round == 0 ? range_of(l) : static_cast<uint32_t>(at >> shift) & (kBins - 1);
      };
      for (int b = tid; b < kBins; b += kThreads) s.count[b] = 0u, s.mass_lo[b] = 0u, s.mass_hi[b] = 0u;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const float l = logit<T>(data + i);
        const uint64_t at = place_of(l, begin + static_cast<uint32_t>(i));
        if (!member(l, at)) continue;
        const uint32_t b = bin_of(l, at);
        if (by_mass) {
          const uint64_t w = Weights::of(weights.exponent(l));
          if (w == 0ull) continue;
          const uint32_t low = static_cast<uint32_t>(w), was = atomicAdd(&s.mass_lo[b], low);
          const uint32_t high = static_cast<uint32_t>(w >> 32) + (was + low < was ? 1u : 0u);
          if (high) atomicAdd(&s.mass_hi[b], high);
        }
        atomicAdd(&s.count[b], 1u);
      }
      cluster_barrier();
      // this CTA's share of the bins, summed over the cluster: kBins / ctas adjacent
      // ones, two a thread where one CTA has them all
      const int share_bins = kBins / p.ctas, mine = share_bins / kThreads > 1 ? share_bins / kThreads : 1;
      uint32_t c[2] = {0u, 0u};
      uint64_t m[2] = {0ull, 0ull};
      const bool has = tid * mine < share_bins;
      const int bin0 = static_cast<int>(rank) * share_bins + tid * mine;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (has && j < mine)
          for (int r = 0; r < p.ctas; ++r) {
            const Shared *o = at_rank(&s, r);
            c[j] += o->count[bin0 + j];
            if (by_mass) m[j] += o->mass_lo[bin0 + j] + (static_cast<uint64_t>(o->mass_hi[bin0 + j]) << 32);
          }
      uint32_t cum_c = c[0] + c[1], total_c;
      uint64_t cum_m = m[0] + m[1], total_m;
      scan(cum_c, cum_m, total_c, total_m, s);
      if (tid == 0) s.part_count = total_c, s.part_mass = total_m;
      cluster_barrier();
      uint32_t all_c = 0;
      uint64_t all_m = 0;
      for (int r = 0; r < p.ctas; ++r) {
        if (r == static_cast<int>(rank)) cum_c += all_c, cum_m += all_m;
        all_c += at_rank(&s, r)->part_count;
        all_m += at_rank(&s, r)->part_mass;
      }
      if (round == 0) {
        if (!by_mass && all_c <= want_count) {
          cluster_barrier();  // the sums are read before the next step writes them
          return;             // fewer tokens than that: the place stays
        }
        // mass before < share * all, in whole units: < ceil(share * all); at least one token
        if (by_mass) target = max(uint64_t{1}, static_cast<uint64_t>(ceil(share * static_cast<double>(all_m))));
      }
      cum_c += before_count;
      cum_m += before_mass;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool hit = by_mass ? (cum_m < target && target <= cum_m + m[j]) : (cum_c < want_count && want_count <= cum_c + c[j]);
        if (has && j < mine && hit)
          for (int r = 0; r < p.ctas; ++r) {
            Shared *o = at_rank(&s, r);
            o->hit_bin = static_cast<uint32_t>(bin0 + j);
            o->hit_count = c[j];
            o->hit_before_count = cum_c;
            o->hit_before_mass = cum_m;
          }
        cum_c += c[j];
        cum_m += m[j];
      }
      cluster_barrier();
      const uint32_t bin = s.hit_bin, inside = s.hit_count;
      before_count = s.hit_before_count;
      before_mass = s.hit_before_mass;
      if (inside <= kList) {
        for (int i = tid; i < n; i += kThreads) {
          const float l = logit<T>(data + i);
          const uint64_t at = place_of(l, begin + static_cast<uint32_t>(i));
          if (!member(l, at) || bin_of(l, at) != bin) continue;
          const uint64_t w = by_mass ? Weights::of(weights.exponent(l)) : 0ull;
          if (by_mass && w == 0ull) continue;
          Shared *o = at_rank(&s, 0);
          const uint32_t k = atomicAdd(&o->list_n, 1u);
          if (k < kList) o->list_at[k] = at, o->list_w[k] = w;
        }
        cluster_barrier();
        if (rank == 0) {
          const int len = static_cast<int>(min(s.list_n, static_cast<uint32_t>(kList)));
          for (int i = tid; i < len; i += kThreads) {
            const uint64_t at = s.list_at[i], w = s.list_w[i];
            uint32_t c0 = before_count;
            uint64_t m0 = before_mass;
            for (int j = 0; j < len; ++j)
              if (s.list_at[j] < at) ++c0, m0 += s.list_w[j];
            if (by_mass ? (m0 < target && target <= m0 + w) : (c0 + 1u == want_count))
              for (int r = 0; r < p.ctas; ++r) at_rank(&s, r)->place = at;
          }
          __syncthreads();
          if (tid == 0) s.list_n = 0u;
        }
        cluster_barrier();
        place = s.place;
        return;
      }
      if (round == 0) range = bin, prefix = 0;
      else prefix = (prefix << 10) | bin;
    }
  };
  if (top_k > 0 && top_k < p.vocab) narrow(false, static_cast<uint32_t>(top_k), 0.0);
  if (top_p < 1.0f) narrow(true, 0u, static_cast<double>(top_p));
  const double least = min_p > 0.0f ? log(static_cast<double>(fminf(min_p, 1.0f))) : -1e300;

  // ---- the draw: weights of adjacent tokens, walked by index ----
  const int per = ((n + kThreads - 1) / kThreads) | 1;  // odd: threads start in different banks
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  auto weight = [&](int i) -> uint64_t {
    const float l = logit<T>(data + i);
    if (!(l > kMinusInf) || place_of(l, begin + static_cast<uint32_t>(i)) > place) return 0ull;
    const double x = weights.exponent(l);
    return x >= least ? Weights::of(x) : 0ull;
  };
  uint64_t sum = 0;
  for (int i = i0; i < i1; ++i) sum += weight(i);
  uint32_t none = 0, none_total;
  uint64_t before = sum, total;
  scan(none, before, none_total, total, s);
  if (tid == 0) s.part_mass = total;
  cluster_barrier();
  uint64_t all = 0, base = 0;
  for (int r = 0; r < p.ctas; ++r) {
    if (r == static_cast<int>(rank)) base = all;
    all += at_rank(&s, r)->part_mass;
  }
  // the first token at which the sum exceeds u * all: its whole part, as sums are whole
  const float u = p.uniform[row];
  double want = u > 0.0f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
  const uint64_t target = min(all - uint64_t{1}, static_cast<uint64_t>(fmin(want, 0x1p63)));
  before += base;
  if (before <= target && target < before + sum) {
    for (int i = i0; i < i1; ++i) {
      before += weight(i);
      if (before > target) {
        p.tokens[row] = static_cast<int64_t>(begin) + i;
        if (p.logprobs)
          p.logprobs[row] = static_cast<float>(weights.exponent(logit<T>(data + i)) -
                                               log(static_cast<double>(all) * (1.0 / kOne)));
        break;
      }
    }
  }
  cluster_barrier();  // no CTA ends while another reads its sums
}

template <typename T>
cudaError_t launch(SampleView p, int rows, int sms, cudaStream_t s) {
  // A row's part in a CTA's shared memory lets two CTAs share an SM, down to
  // 4096 tokens a CTA while there are SMs without one.
  constexpr int kMost = 96 * 1024 / sizeof(T);
  p.ctas = 1;
  while (p.ctas < 8 && ((p.vocab + p.ctas - 1) / p.ctas > kMost ||
                        (static_cast<int64_t>(rows) * p.ctas < 2 * sms && p.vocab / p.ctas >= 2 * 4096)))
    p.ctas *= 2;
  p.slice = (p.vocab + p.ctas - 1) / p.ctas;
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + 16 + static_cast<size_t>(p.slice) * sizeof(T);
  cudaError_t e = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * static_cast<unsigned>(p.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, k_sample<T>, p);
}

bool misaligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

}  // namespace

int sample(const FnSampleArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (a->logits_dtype > FNMOE_DTYPE_F32) { err = "logits must be bfloat16 or float32"; return FNMOE_ERR_UNSUPPORTED; }
  if (a->vocab == 0 || a->vocab > FNMOE_SAMPLE_MAX_VOCAB) {
    err = "vocab must be between 1 and " + std::to_string(FNMOE_SAMPLE_MAX_VOCAB);
    return FNMOE_ERR_SHAPE;
  }
  if (a->rows > 0x0FFFFFFFu) { err = "at most 2^28 - 1 rows"; return FNMOE_ERR_SHAPE; }
  if (a->rows == 0) return FNMOE_OK;
  if (!a->logits || !a->uniform || !a->tokens) { err = "logits, uniform and tokens are required"; return FNMOE_ERR_NULL; }
  if (a->rows > 1 && a->logits_stride < a->vocab) { err = "logits_stride must cover a row"; return FNMOE_ERR_SHAPE; }
  if (misaligned(a->logits, a->logits_dtype == FNMOE_DTYPE_F32 ? 4 : 2) || misaligned(a->uniform, 4) ||
      misaligned(a->temperatures, 4) || misaligned(a->top_ks, 4) || misaligned(a->top_ps, 4) ||
      misaligned(a->min_ps, 4) || misaligned(a->tokens, 8) || misaligned(a->logprobs, 4)) {
    err = "arrays must be aligned to their elements";
    return FNMOE_ERR_VALUE;
  }
  SampleView p{};
  p.logits = a->logits;
  p.uniform = a->uniform;
  p.temperatures = a->temperatures;
  p.top_ks = a->top_ks;
  p.top_ps = a->top_ps;
  p.min_ps = a->min_ps;
  p.tokens = a->tokens;
  p.logprobs = a->logprobs;
  p.stride = a->logits_stride;
  p.vocab = static_cast<int>(a->vocab);
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  const int sms = device_info().sms, rows = static_cast<int>(a->rows);
  cudaError_t e = a->logits_dtype == FNMOE_DTYPE_F32 ? launch<float>(p, rows, sms, s) : launch<uint16_t>(p, rows, sms, s);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return FNMOE_OK;
  err = std::string("sample: ") + cudaGetErrorString(e);
  return FNMOE_ERR_LAUNCH;
}

}  // namespace fnmoe
