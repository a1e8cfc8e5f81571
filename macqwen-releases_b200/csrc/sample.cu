// sample.cu -- one token a row of logits by temperature, top-k, top-p and min-p
// from a given uniform number, in one launch that reads the logits once.
//
// Ranked by falling logit, equal ones by rising index, each filter keeps a
// prefix, so together they keep the tokens up to one place: a (logit, index)
// pair, found by counting instead of sorting.  The row lies in the shared
// memory of a cluster's CTAs; a histogram of the logits (1024 equal ranges)
// names the range in which the place falls.  Where that range and those above
// hold few tokens (top_k up to about a thousand, a nucleus of as many), they are
// gathered in one CTA, which sorts them and does the rest.  Otherwise the
// tokens of the range alone are gathered and ranked; a range that holds too
// many of them (ties, outliers) is divided again, by the bits of (logit,
// index), until it does not; and the draw walks the whole row by index.
//
// Weights are 2^((l - max) log2(e) / T) in float64, held as integers of 2^-44 of
// the largest: sums are then exact and do not depend on the order of threads or
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
constexpr uint64_t kAll = ~0ull;  // past every place
constexpr uint64_t kOne = 1ull << 44;  // the largest weight
constexpr int kRoots = 128;
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
  uint32_t count[kBins];                   // this CTA's histogram
  uint32_t mass_lo[kBins], mass_hi[kBins]; // and its weights
  uint64_t list_at[kList], list_w[kList];  // (rank 0) gathered tokens: places and weights
  double root[kRoots];                     // 2^(j / kRoots)
  uint64_t warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  float warp_max[kWarps], warp_min[kWarps];
  float row_max, row_min;                  // of this CTA's part
  uint64_t part_mass;                      // of this CTA's kept tokens
  uint32_t list_n;                         // (rank 0)
  uint32_t best;                           // this CTA's lowest index of the largest logit
  // the range in which the place falls
  uint32_t hit_bin, hit_count, hit_before_count;
  uint64_t hit_before_mass;
  uint64_t place;                          // the last kept token (written to every copy by rank 0)
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
__device__ __forceinline__ float logit_at(uint64_t place) {
  const uint32_t up = ~static_cast<uint32_t>(place >> kIndexBits);
  return __uint_as_float((up & 0x80000000u) ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ uint32_t index_at(uint64_t place) {
  return static_cast<uint32_t>(place) & ((1u << kIndexBits) - 1u);
}

// A row's weights in units of 2^-44 of the largest.
struct Weights {
  float top, low;       // the largest logit; what does not lie above `low` weighs less than half a unit
  double per;           // log2(e) / temperature
  const double *root;
  __device__ __forceinline__ double exponent(float l) const {
    return (static_cast<double>(l) - static_cast<double>(top)) * per;
  }
  // 2^y for -46 < y <= 0, to 2^-49 of itself: y = k + j / 128 + r, 2^r by its
  // series up to r^4 (the next term is below 2^-49), 2^(j / 128) from the
  // table, 2^(k + 44) in the exponent; adding 2^52 leaves the nearest whole
  // number in the low bits.  (CUDA's exp would be three times the float64
  // operations.)
  __device__ __forceinline__ uint64_t power(double y) const {
    constexpr double kRound = 0x1.8p45;  // its last bit is 2^-7
    const double t = __dadd_rn(y, kRound), r = __dadd_rn(y, -__dadd_rn(t, -kRound));
    const int m = __double2loint(t);
    double q = fma(r, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0c0p-5);  // ln(2)^4 / 24, ln(2)^3 / 6
    q = fma(r, q, 0x1.ebfbdff82c58fp-3);                            // ln(2)^2 / 2
    q = fma(r, q, 0x1.62e42fefa39efp-1);                            // ln(2)
    q = fma(r, q, 1.0);
    const double s = root[m & (kRoots - 1)];
    const double scaled = __hiloint2double(__double2hiint(s) + (((m >> 7) + 44) << 20), __double2loint(s));
    return static_cast<uint64_t>(__double_as_longlong(fma(q, scaled, 0x1p52))) & ((1ull << 52) - 1ull);
  }
  __device__ __forceinline__ uint64_t of(float l) const {
    if (l == top) return kOne;
    return l > low ? power(exponent(l)) : 0ull;
  }
  // Four at once, whose chains of float64 operations overlap; 0 where `on` is
  // false or log2 of the weight (of the largest) is below `least`.
  __device__ __forceinline__ void of4(const float (&l)[4], const bool (&on)[4], double least, uint64_t (&w)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool some = on[e] && (l[e] > low || l[e] == top);
      const double y = l[e] == top ? 0.0 : exponent(l[e]);
      w[e] = power(some ? y : 0.0);
      if (!some || y < least) w[e] = 0ull;
    }
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

// Sorts s.list_at[0 .. len), a power of two up to kList, upwards.
__device__ void sort_list(Shared &s, int len) {
  for (int size = 2; size <= len; size <<= 1)
    for (int gap = size >> 1; gap > 0; gap >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < len / 2; i += kThreads) {
        const int a = 2 * i - (i & (gap - 1)), b = a + gap;  // a: the pairs' first ones, gap bit clear
        const uint64_t x = s.list_at[a], y = s.list_at[b];
        if ((x > y) == ((a & size) == 0)) s.list_at[a] = y, s.list_at[b] = x;
      }
    }
  __syncthreads();
}

struct Settings {
  float t, top_p, min_p, u;
  int top_k;  // 0: off
};

// The whole part of u times `all`, below all: the draw is the first token at
// which the sum exceeds u * all, and sums are whole.
__device__ __forceinline__ uint64_t drawn_at(float u, uint64_t all) {
  const double want = u > 0.0f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
  return min(all - uint64_t{1}, static_cast<uint64_t>(fmin(want, 0x1p63)));
}

__device__ __forceinline__ void write_row(const SampleView &p, int row, uint32_t index, float l, const Weights &weights,
                                          float t, uint64_t all) {
  p.tokens[row] = static_cast<int64_t>(index);
  if (p.logprobs) {
    const double x = l == weights.top ? 0.0 : (static_cast<double>(l) - static_cast<double>(weights.top)) / static_cast<double>(t);
    p.logprobs[row] = static_cast<float>(x - log(static_cast<double>(all) * (1.0 / kOne)));
  }
}

// The rest of a row whose every token that may be kept is in rank 0's list, by
// that CTA.  by_count: the list holds the first top_k, and more; else what may
// be kept by top-p, the weights before a kept token staying below `target`.
__device__ void draw_from_list(const SampleView &p, int row, const Settings &set, const Weights &weights, double least,
                               bool by_count, uint64_t target, Shared &s) {
  const int tid = threadIdx.x, n = static_cast<int>(s.list_n);
  int len = 2;
  while (len < n) len <<= 1;
  for (int i = n + tid; i < len; i += kThreads) s.list_at[i] = kAll;
  sort_list(s, len);
  // threads take two adjacent tokens by rank
  const int kept_n = by_count ? min(set.top_k, n) : n;
  uint64_t at[2], w[2];
  float l[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = 2 * tid + j;
    at[j] = e < kept_n ? s.list_at[e] : kAll;
    l[j] = logit_at(at[j]);
    w[j] = e < kept_n ? weights.of(l[j]) : 0ull;
  }
  uint32_t none = 0, none_total;
  uint64_t before = w[0] + w[1], total;
  scan(none, before, none_total, total, s);
  if (by_count)
    target = set.top_p < 1.0f ? max(uint64_t{1}, static_cast<uint64_t>(ceil(static_cast<double>(set.top_p) * static_cast<double>(total)))) : kAll;
  uint64_t kept[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const bool keep = before < target && (l[j] == weights.top || weights.exponent(l[j]) >= least);
    before += w[j];
    const int e = 2 * tid + j;
    if (!keep) w[j] = 0ull;
    // by index now, with the rank behind it; tokens of no weight are not drawn
    kept[j] = w[j] != 0ull ? (static_cast<uint64_t>(index_at(at[j])) << 10) | static_cast<uint64_t>(e) : kAll;
    if (e < len) s.list_at[e] = kept[j], s.list_w[e] = w[j];  // list_at[e] was read by this thread alone since the sort
  }
  sort_list(s, len);
  uint64_t key[2], v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = 2 * tid + j;
    key[j] = e < len ? s.list_at[e] : kAll;
    v[j] = key[j] != kAll ? s.list_w[key[j] & (kList - 1)] : 0ull;
  }
  before = v[0] + v[1];
  scan(none, before, none_total, total, s);
  const uint64_t drawn = drawn_at(set.u, total);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (before <= drawn && drawn < before + v[j]) {
      s.hit_bin = static_cast<uint32_t>(key[j]) & (kList - 1);
    }
    before += v[j];
  }
  __syncthreads();
  // the drawn token's logit, by the thread that had it by rank
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (s.hit_bin == static_cast<uint32_t>(2 * tid + j)) write_row(p, row, index_at(at[j]), l[j], weights, set.t, total);
}

// One row, in a cluster of p.ctas CTAs.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(SampleView p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.ctas;
  const uint32_t rank = blockIdx.x % p.ctas;
  const uint32_t begin = rank * static_cast<uint32_t>(p.slice);
  const int n = max(0, min(p.slice, p.vocab - static_cast<int>(begin)));
  if (tid < kRoots) s.root[tid] = exp2(static_cast<double>(tid) / kRoots);
  if (tid == 0) s.list_n = 0u, s.best = 0xFFFFFFFFu;
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
  // the logits of a vector, in order
  auto unpack = [&](uint4 v, auto &&f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        f(__uint_as_float(w[e]), e);
      } else {
        f(__uint_as_float(w[e] << 16), 2 * e);
        f(__uint_as_float(w[e] & 0xFFFF0000u), 2 * e + 1);
      }
    }
  };
  auto take = [&](uint4 v, int i) {
    data4[i] = v;
    unpack(v, [&](float l, int) { meet(l); });
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
  // every token of the part, from shared memory: f(four logits, index of the
  // first in the part); places without a token hold -infinity
  auto each4 = [&](auto &&f) {
    auto one = [&](int i) {
      const float l[4] = {logit<T>(data + i), kMinusInf, kMinusInf, kMinusInf};
      f(l, i);
    };
    if (tid < head) one(tid);
    for (int i = tid; i < vecs; i += kThreads) {
      float l[kVec];
      unpack(data4[i], [&](float x, int e) { l[e] = x; });
#pragma unroll
      for (int g = 0; g < kVec; g += 4) {
        const float l4[4] = {l[g], l[g + 1], l[g + 2], l[g + 3]};
        f(l4, head + i * kVec + g);
      }
    }
    const int tail = head + vecs * kVec;
    if (tail + tid < n) one(tail + tid);
  };
  auto each = [&](auto &&f) {
    each4([&](const float (&l)[4], int i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(l[e], i + e);
    });
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
  }
  if (lane == 0) s.warp_max[warp] = hi, s.warp_min[warp] = lo;
  // the row's settings
  Settings set;
  set.t = p.temperatures ? p.temperatures[row] : p.temperature;
  set.top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  set.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  set.min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  set.u = p.uniform[row];
  if (set.top_k < 0 || set.top_k >= p.vocab) set.top_k = p.vocab == 1 ? 1 : 0;
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
  const Weights weights{hi, __fsub_rd(hi, __fmul_ru(set.t, 31.54f)), 1.4426950408889634074 / static_cast<double>(set.t), s.root};
  // the largest logit: asked for, or all that there is
  if (!(set.t > 0.0f) || set.top_k == 1 || !(set.top_p > 0.0f) || !(hi > kMinusInf)) {
    uint32_t best = 0xFFFFFFFFu;
    if (hi > kMinusInf)
      each([&](float l, int i) {
        if (l == hi) best = min(best, begin + static_cast<uint32_t>(i));
      });
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
  const double least = set.min_p > 0.0f ? log2(static_cast<double>(fminf(set.min_p, 1.0f))) : -1e300;

  // ---- the place of the last kept token ----
  float cut = kMinusInf;  // its logit and its index: so far every token that is not masked
  int cut_index = -1;
  auto kept = [&](float l, int i) { return l > cut || (l == cut && static_cast<int>(begin) + i <= cut_index); };
  // Tokens up to there: the first set.top_k of them, or (by_mass)
  // those before whose place less than set.top_p of their weights lies.  True:
  // every token that may be kept went to rank 0's list instead.
  auto narrow = [&](const bool by_mass, uint64_t &target) {
    const uint32_t want = static_cast<uint32_t>(set.top_k);
    // ranges of the first round: equal parts of the logits that can matter
    float span = __fsub_rn(hi, lo);
    if (by_mass) span = fminf(span, __fsub_rn(hi, weights.low));
    const float per = span > 0.0f ? __fdiv_rn(static_cast<float>(kBins), span) : 0.0f;
    auto range_of = [&](float l) {  // rises (weakly) with falling logits
      const int b = static_cast<int>(__fmul_rn(__fsub_rn(hi, l), per));
      return static_cast<uint32_t>(min(max(b, 0), kBins - 1));
    };
    auto append = [&](uint64_t at, uint64_t w) {
      Shared *o = at_rank(&s, 0);
      const uint32_t k = atomicAdd(&o->list_n, 1u);
      if (k < kList) o->list_at[k] = at, o->list_w[k] = w;
    };
    uint32_t range = 0;   // chosen in the first round
    uint64_t prefix = 0;  // of (logit, index), chosen in later rounds
    uint32_t before_count = 0;
    uint64_t before_mass = 0;
    for (int round = 0;; ++round) {
      const int shift = kPlaceBits - 10 * round;  // of the later rounds' digits: 40, 30, .., 0
      // the bin of a kept token, or kBins where an earlier round left it out
      auto bin_of = [&](float l, int i) {
        const uint32_t r = range_of(l);
        if (round == 0) return r;
        const uint64_t at = place_of(l, begin + static_cast<uint32_t>(i));
        if (r != range || (round > 1 && (at >> (shift + 10)) != prefix)) return static_cast<uint32_t>(kBins);
        return static_cast<uint32_t>(at >> shift) & (kBins - 1);
      };
      for (int b = tid; b < kBins; b += kThreads) s.count[b] = 0u, s.mass_lo[b] = 0u, s.mass_hi[b] = 0u;
      __syncthreads();
      each4([&](const float (&l)[4], int i) {
        bool on[4];
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          on[e] = kept(l[e], i + e);
          b[e] = on[e] ? bin_of(l[e], i + e) : kBins;
          on[e] = b[e] < kBins;
        }
        if (by_mass) {
          uint64_t w[4];
          weights.of4(l, on, -1e300, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (w[e] == 0ull) continue;
            atomicAdd(&s.count[b[e]], 1u);
            const uint32_t low = static_cast<uint32_t>(w[e]), was = atomicAdd(&s.mass_lo[b[e]], low);
            const uint32_t high = static_cast<uint32_t>(w[e] >> 32) + (was + low < was ? 1u : 0u);
            if (high) atomicAdd(&s.mass_hi[b[e]], high);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (on[e]) atomicAdd(&s.count[b[e]], 1u);
        }
      });
      cluster_barrier();
      // the cluster's histogram, two bins a thread, summed by every CTA for itself
      uint32_t c[2] = {0u, 0u};
      uint64_t m[2] = {0ull, 0ull};
      for (int r = 0; r < p.ctas; ++r) {
        const Shared *o = at_rank(&s, r);
        const uint2 k = reinterpret_cast<const uint2 *>(o->count)[tid];
        c[0] += k.x, c[1] += k.y;
        if (by_mass) {
          const uint2 a = reinterpret_cast<const uint2 *>(o->mass_lo)[tid], b = reinterpret_cast<const uint2 *>(o->mass_hi)[tid];
          m[0] += a.x + (static_cast<uint64_t>(b.x) << 32), m[1] += a.y + (static_cast<uint64_t>(b.y) << 32);
        }
      }
      uint32_t cum_c = c[0] + c[1], all_c;
      uint64_t cum_m = m[0] + m[1], all_m;
      scan(cum_c, cum_m, all_c, all_m, s);
      if (round == 0) {
        if (!by_mass && all_c <= want) {
          cluster_barrier();  // the histograms are read before they are cleared again
          return false;       // no more tokens than that: all stay
        }
        // mass before < top_p * all, in whole units: < ceil(top_p * all); at least one token
        if (by_mass) target = max(uint64_t{1}, static_cast<uint64_t>(ceil(static_cast<double>(set.top_p) * static_cast<double>(all_m))));
      }
      cum_c += before_count;
      cum_m += before_mass;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (by_mass ? (cum_m < target && target <= cum_m + m[j]) : (cum_c < want && want <= cum_c + c[j])) {
          s.hit_bin = static_cast<uint32_t>(2 * tid + j);
          s.hit_count = c[j];
          s.hit_before_count = cum_c;
          s.hit_before_mass = cum_m;
        }
        cum_c += c[j];
        cum_m += m[j];
      }
      __syncthreads();
      const uint32_t bin = s.hit_bin, inside = s.hit_count;
      before_count = s.hit_before_count;
      before_mass = s.hit_before_mass;
      if (round == 0 && before_count + inside <= kList) {
        each([&](float l, int i) {
          if (kept(l, i) && range_of(l) <= bin && (!by_mass || weights.of(l) != 0ull))
            append(place_of(l, begin + static_cast<uint32_t>(i)), 0ull);
        });
        cluster_barrier();
        return true;
      }
      if (inside <= kList) {
        each([&](float l, int i) {
          if (!kept(l, i) || bin_of(l, i) != bin) return;
          const uint64_t w = by_mass ? weights.of(l) : 0ull;
          if (!by_mass || w != 0ull) append(place_of(l, begin + static_cast<uint32_t>(i)), w);
        });
        cluster_barrier();
        if (rank == 0) {
          const int len = static_cast<int>(min(s.list_n, static_cast<uint32_t>(kList)));
          for (int i = tid; i < len; i += kThreads) {
            const uint64_t at = s.list_at[i], w = s.list_w[i];
            uint32_t c0 = before_count;
            uint64_t m0 = before_mass;
            for (int j = 0; j < len; ++j)
              if (s.list_at[j] < at) ++c0, m0 += s.list_w[j];
            if (by_mass ? (m0 < target && target <= m0 + w) : (c0 + 1u == want))
              for (int r = 0; r < p.ctas; ++r) at_rank(&s, r)->place = at;
          }
          __syncthreads();
          if (tid == 0) s.list_n = 0u;
        }
        cluster_barrier();
        cut = logit_at(s.place);
        cut_index = static_cast<int>(index_at(s.place));
        return false;
      }
      cluster_barrier();  // the histograms are read before they are cleared again
      if (round == 0) range = bin, prefix = 0;
      else prefix = (prefix << 10) | bin;
    }
  };
  uint64_t target = 0;
  const bool by_count = set.top_k > 0 && narrow(false, target);
  if (by_count || (set.top_p < 1.0f && narrow(true, target))) {
    if (rank == 0) draw_from_list(p, row, set, weights, least, by_count, target, s);
    return;  // nobody reads the others' shared memory any more
  }

  // ---- the draw: weights of adjacent tokens, walked by index ----
  const int per = ((n + kThreads - 1) / kThreads) | 1;  // odd: threads start in different banks
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  auto weigh = [&](int i, uint64_t (&w)[4]) {  // four tokens from i on, none from i1 on
    float l[4];
    bool on[4], some = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      l[e] = i + e < i1 ? logit<T>(data + i + e) : kMinusInf;
      on[e] = kept(l[e], i + e);
      some |= on[e];
      w[e] = 0ull;
    }
    if (some) weights.of4(l, on, least, w);
  };
  uint64_t sum = 0, w4[4];
  for (int i = i0; i < i1; i += 4) {
    weigh(i, w4);
    sum += (w4[0] + w4[1]) + (w4[2] + w4[3]);
  }
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
  const uint64_t drawn = drawn_at(set.u, all);
  before += base;
  if (before <= drawn && drawn < before + sum) {
    for (int i = i0; i < i1 && before <= drawn; i += 4) {
      weigh(i, w4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (before <= drawn && drawn < before + w4[e])
          write_row(p, row, begin + static_cast<uint32_t>(i + e), logit<T>(data + i + e), weights, set.t, all);
        before += w4[e];
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
