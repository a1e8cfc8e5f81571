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
//
// Bound by issue slots (57 to 163 instructions a token over all passes) and, for
// few rows, by short steps that follow one another (loads, the largest and its
// barriers 3.6 us, then the bound's search, a list, its ranks and sums): 1 x 131072
// with top-k 50, top-p and min-p 10.2 us; 64 x 131072 33.4 us, with settings of
// their own 55 us, top-p alone 78 us.
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
constexpr int kList = 512;        // tokens of a range that are ranked against one another
constexpr int kFew = 384;         // kept tokens that one CTA finishes by itself
constexpr int kGroups = 256;      // groups of tokens whose maxima bound the top-k ..
constexpr int kByGroups = 190;    // .. up to this k: about 256 ln(1 / (1 - k / 256)) tokens lie above the bound
constexpr int kBlock = 512;       // adjacent tokens whose weights are summed together for the draw
constexpr int kMaxBlocks = 128;
constexpr int kMaxCtas = 16;
constexpr int kRoots = 512;
constexpr int kIndexBits = 18;    // FNMOE_SAMPLE_MAX_VOCAB
constexpr int kPlaceBits = 32 + kIndexBits;
constexpr uint64_t kAll = ~0ull;  // past every place
constexpr uint64_t kOne = 1ull << 44;  // the largest weight
constexpr float kMinusInf = -__builtin_inff();
constexpr int kEvery = 0x7FFFFFFF;

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

// A CTA's working memory.  What other CTAs have to know is written into their
// copies before a cluster barrier, so that it is read near by after it.
struct Shared {
  union {
    struct {
      uint32_t count[kBins];                     // this CTA's histogram (read by the others)
      uint32_t mass_lo[kBins], mass_hi[kBins];   // and its weights
    };
    struct {
      uint64_t pulled[kList], pulled_w[kList];   // (rank 0) the cluster's gathered tokens, and their weights
    };
  };
  union {
    struct {
      uint32_t count[kBins];                     // the cluster's histogram
      uint64_t mass[kBins];
    } sum;
    struct {
      uint64_t at[kList], w[kList];              // gathered tokens: places and weights (read by rank 0)
    } list;
    float pack[kWarps][kBlock / 2];              // the draw: a warp's kept logits
  };
  double root[kRoots];                           // 2^(44 + j / kRoots)
  uint64_t block_mass[kMaxBlocks];
  float own_group[kGroups], group[kGroups];      // largest logits of groups: this CTA's, the cluster's
  uint64_t warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  float warp_max[kWarps], warp_min[kWarps];
  float rank_max[kMaxCtas], rank_min[kMaxCtas];
  uint64_t rank_mass[kMaxCtas];
  uint32_t rank_list[kMaxCtas];
  uint32_t list_n;
  uint32_t best;                                 // (rank 0) lowest index of the largest logit
  float bound;                                   // no more than the top_k-th largest logit
  // the range in which the place falls
  uint32_t hit_bin, hit_count, hit_before_count;
  uint64_t hit_before_mass;
  uint64_t place;                                // the last kept token (written to every copy by rank 0)
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
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
  // The weight of a logit in (low, top]: 2^y, y = (l - top) per = k + j / 512 + r,
  // to 2^-46 of itself: 2^r by its series up to r^3, 2^(44 + j / 512) from the
  // table, 2^k in the exponent; adding 2^52 leaves the nearest whole number in the
  // low bits.  Eight float64 operations; CUDA's exp takes three times that.
  __device__ __forceinline__ uint64_t of(float l) const {
    constexpr double kRound = 0x1.8p43;  // its last bit is 2^-9
    const double d = l == top ? 0.0 : static_cast<double>(l) - static_cast<double>(top);
    const double t = fma(d, per, kRound);
    const double r = fma(d, per, -__dadd_rn(t, -kRound));
    const int m = __double2loint(t);
    double q = fma(r, 0x1.c6b08d704a0c0p-5, 0x1.ebfbdff82c58fp-3);  // ln(2)^3 / 6, ln(2)^2 / 2
    q = fma(r, q, 0x1.62e42fefa39efp-1);                            // ln(2)
    q = fma(r, q, 1.0);
    const double s = root[m & (kRoots - 1)];
    const double scaled = __hiloint2double(__double2hiint(s) + static_cast<int>(static_cast<uint32_t>(m) << 11 & 0xFFF00000u), __double2loint(s));
    return static_cast<uint64_t>(__double_as_longlong(fma(q, scaled, 0x1p52))) & ((1ull << 52) - 1ull);
  }
  __device__ __forceinline__ uint64_t any(float l) const { return l > low || l == top ? of(l) : 0ull; }
};

// What is kept: logits above `l`, and those equal to it up to index `index`.
struct Cut {
  float l;
  int index;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > l || (x == l && i <= index); }
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
// The units that the weights before a kept token stay below, for top-p of `all`.
__device__ __forceinline__ uint64_t share_of(float top_p, uint64_t all) {
  return max(uint64_t{1}, static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(all))));
}

__device__ __forceinline__ void write_row(const SampleView &p, int row, uint32_t index, float l, const Weights &weights,
                                          uint64_t all) {
  p.tokens[row] = static_cast<int64_t>(index);
  if (p.logprobs) {
    const double x = l == weights.top ? 0.0 : weights.exponent(l) * 0.6931471805599453094;
    p.logprobs[row] = static_cast<float>(x - log(static_cast<double>(all) * (1.0 / kOne)));
  }
}

// The rest of a row whose every token that may be kept is among rank 0's n
// pulled ones (n <= kFew), by that CTA.  by_count: they hold the
// first top_k, and more; else what may be kept by top-p, the weights before a
// kept token staying below `target`.  The two orders that this needs, by rank
// for the filters and by index for the draw, come from counting what lies before.
__device__ void draw_from_list(const SampleView &p, int row, const Settings &set, const Weights &weights, double least,
                               bool by_count, uint64_t target, int n, Shared &s) {
  const int tid = threadIdx.x;
  // adjacent threads of a token share what is counted for it
  int team = 1;
  while (team < 32 && 2 * team * n <= kThreads) team *= 2;
  const int token = tid / team, part = tid % team;
  {
    const uint64_t mine = token < n ? s.pulled[token] : 0ull;
    int r = 0;
    if (token < n) {
#pragma unroll 4
      for (int j = part; j < n; j += team) r += s.pulled[j] < mine;
    }
    for (int o = 1; o < team; o <<= 1) r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
    if (token < n && part == 0) s.list.at[r] = mine;
  }
  __syncthreads();
  const int kept_n = by_count ? min(set.top_k, n) : n;
  const uint64_t at = tid < kept_n ? s.list.at[tid] : kAll;
  const float l = logit_at(at);
  uint64_t w = tid < kept_n ? weights.any(l) : 0ull;
  uint32_t none = 0, none_total;
  uint64_t before = w, total;
  scan(none, before, none_total, total, s);
  if (by_count) target = set.top_p < 1.0f ? share_of(set.top_p, total) : kAll;
  if (!(before < target && (l == weights.top || weights.exponent(l) >= least))) w = 0ull;
  if (tid < n) s.pulled[tid] = at, s.list.w[tid] = w;
  uint64_t sum = w;
  scan(none, sum, none_total, total, s);
  const uint64_t drawn = drawn_at(set.u, total);
  const uint64_t held = token < n ? s.list.w[token] : 0ull, mine = token < n ? s.pulled[token] : 0ull;
  const uint32_t index = index_at(mine);
  uint64_t lower = 0;
  if (held != 0ull) {
#pragma unroll 4
    for (int j = part; j < n; j += team) lower += index_at(s.pulled[j]) < index ? s.list.w[j] : 0ull;
  }
  for (int o = 1; o < team; o <<= 1) lower += __shfl_xor_sync(0xFFFFFFFFu, lower, o);
  if (part == 0 && lower <= drawn && drawn < lower + held) write_row(p, row, index, logit_at(mine), weights, total);
}

// The least float, in the order of place_of, at or below `most` for which `above`
// holds; `above` rises with it and holds for `most`.  By its bits, five at a time:
// a lane a candidate (a whole warp calls it).
template <typename F>
__device__ __forceinline__ float least_float(float most, F &&above) {
  const uint32_t lane = threadIdx.x & 31, end = ~static_cast<uint32_t>(place_of(most, 0) >> kIndexBits);
  uint32_t below = 0u;  // the largest for which it does not hold, as far as it is known
#pragma unroll 1
  for (int shift = 27; shift > -5; shift -= 5) {
    const uint32_t key = below | (shift >= 0 ? lane << shift : lane >> -shift);
    const float x = __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
    // what is not a number sorts below -infinity: no; above infinity: past `most`
    const uint32_t less = __ballot_sync(0xFFFFFFFFu, !(key >= end || (x >= kMinusInf && above(x))));
    below = __shfl_sync(0xFFFFFFFFu, key, 31 - __clz(less));  // lane 0 is always among them
  }
  const uint32_t first = below + 1u;
  return __uint_as_float((first & 0x80000000u) ? first & 0x7FFFFFFFu : ~first);
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
  static_assert(kRoots == kThreads, "a root a thread");
  s.root[tid] = exp2(44.0 + static_cast<double>(tid) / kRoots);
  if (tid == 0) s.list_n = 0u, s.best = 0xFFFFFFFFu;
  cluster_arrive();  // this CTA is here: the others wait for it before they write into its memory
  pdl_wait();
  pdl_trigger();
  // the row's settings
  Settings set;
  set.t = p.temperatures ? p.temperatures[row] : p.temperature;
  set.top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  set.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  set.min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  set.u = p.uniform[row];

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
  const int head = min(n, (kVec - skew) % kVec), vecs = (n - head) / kVec, tail = head + vecs * kVec;
  if (tid < head) {
    data[tid] = src[tid];
    meet(logit<T>(src + tid));
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
  if (tail + tid < n) {
    data[tail + tid] = src[tail + tid];
    meet(logit<T>(src + tail + tid));
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
    if (tail + tid < n) one(tail + tid);
  };
  // groups of 2 ctas threads, so that a cluster has kGroups of them
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
    if (o == p.ctas && lane % (2 * o) == 0) s.own_group[tid / (2 * o)] = hi;
  }
  if (lane == 0) s.warp_max[warp] = hi, s.warp_min[warp] = lo;
  if (set.top_k < 0 || set.top_k >= p.vocab) set.top_k = 0;
  const bool by_groups = set.top_k > 1 && set.top_k <= kByGroups;
  __syncthreads();
  cluster_wait();
  if (by_groups && tid < kGroups) {
    const int each = kGroups / p.ctas;
    at_rank(&s, tid / each)->group[rank * each + tid % each] = s.own_group[tid % each];
  }
  if (warp == 0) {
    hi = s.warp_max[lane % kWarps], lo = s.warp_min[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
    }
    if (lane < p.ctas) {
      Shared *o = at_rank(&s, lane);
      o->rank_max[rank] = hi;
      o->rank_min[rank] = lo;
    }
  }
  cluster_barrier();
  hi = kMinusInf, lo = -kMinusInf;
  for (int r = 0; r < p.ctas; ++r) {
    hi = fmaxf(hi, s.rank_max[r]);
    lo = fminf(lo, s.rank_min[r]);
  }
  // the largest logit: asked for, or all that there is
  if (!(set.t > 0.0f) || set.top_k == 1 || !(set.top_p > 0.0f) || !(hi > kMinusInf)) {
    uint32_t best = 0xFFFFFFFFu;
    if (hi > kMinusInf)
      each4([&](const float (&l)[4], int i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (l[e] == hi) best = min(best, begin + static_cast<uint32_t>(i + e));
      });
    best = __reduce_min_sync(0xFFFFFFFFu, best);
    if (lane == 0 && best != 0xFFFFFFFFu) atomicMin(&at_rank(&s, 0)->best, best);
    cluster_barrier();
    if (rank == 0 && tid == 0) {
      p.tokens[row] = s.best == 0xFFFFFFFFu ? -1 : static_cast<int64_t>(s.best);
      if (p.logprobs) p.logprobs[row] = 0.0f;
    }
    return;
  }
  const Weights weights{hi, hi < -kMinusInf ? __fsub_rd(hi, __fmul_ru(set.t, 31.54f)) : hi, 1.4426950408889634074 / static_cast<double>(set.t), s.root};
  const double least = set.min_p > 0.0f ? log2(static_cast<double>(fminf(set.min_p, 1.0f))) : -1e300;

  // ---- the place of the last kept token ----
  Cut cut{kMinusInf, -1};  // so far every token that is not masked
  // of the tokens that `c` keeps, those that weigh something
  auto weighing = [&](Cut c) {
    if (weights.low >= hi) return c.l < hi ? Cut{hi, kEvery} : c;
    return weights.low >= c.l ? Cut{weights.low, -1} : c;
  };
  auto append = [&](uint64_t at, uint64_t w) {
    const uint32_t k = atomicAdd(&s.list_n, 1u);
    if (k < kList) s.list.at[k] = at, s.list.w[k] = w;
  };
  // The number of tokens in the cluster's lists.
  auto listed = [&]() {
    __syncthreads();
    if (tid < p.ctas) at_rank(&s, tid)->rank_list[rank] = s.list_n;
    cluster_barrier();
    uint32_t all = 0;
    for (int r = 0; r < p.ctas; ++r) all += s.rank_list[r];
    return all;
  };
  // Rank 0 takes them, up to kList.
  auto pull = [&]() {
    int from = 0, r = 0;
    for (int i = tid; i < kList; i += kThreads) {
      while (r < p.ctas && i >= from + static_cast<int>(s.rank_list[r])) from += static_cast<int>(s.rank_list[r++]);
      if (r == p.ctas) break;
      const Shared *o = at_rank(&s, r);
      s.pulled[i] = o->list.at[i - from];
      s.pulled_w[i] = o->list.w[i - from];
    }
    __syncthreads();
  };
  // Tokens up to there: the first set.top_k of them, or (by_mass) those before
  // whose place less than set.top_p of their weights lies.  Not 0: every token
  // that may be kept is in the cluster's lists instead, so many of them.
  auto narrow = [&](const bool by_mass, uint64_t &target) {
    const uint32_t want = static_cast<uint32_t>(set.top_k);
    const Cut among = by_mass ? weighing(cut) : cut;
    // ranges of the first round: equal parts of the logits that can matter
    float span = fminf(__fsub_rn(hi, lo), 0x1p127f);
    if (by_mass) span = fminf(span, __fsub_rn(hi, weights.low));
    // (Logits that lie closer than 2^-100 share a range, and the digits divide
    // it: the quotient stays finite, so that ranges always rise.)
    span = fmaxf(span, 0x1p-100f);
    const float per = __fdiv_rn(static_cast<float>(kBins - 1), span);
    // 2^23 and the range, the nearest whole number, which rises (weakly) with
    // falling logits; where the largest is infinite all are in the last one
    auto spot = [&](float l) { return fmaf(fminf(__fsub_rn(hi, l), span), per, 0x1p23f); };
    auto range_of = [&](float l) { return __float_as_uint(spot(l)) & (kBins - 1); };
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
        uint32_t b[4];
        uint64_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          b[e] = among.keeps(l[e], static_cast<int>(begin) + i + e) ? bin_of(l[e], i + e) : kBins;
          if (by_mass) w[e] = weights.of(b[e] < kBins ? l[e] : hi);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (b[e] >= kBins) continue;
          atomicAdd(&s.count[b[e]], 1u);
          if (by_mass) {
            const uint32_t low = static_cast<uint32_t>(w[e]), was = atomicAdd(&s.mass_lo[b[e]], low);
            const uint32_t high = static_cast<uint32_t>(w[e] >> 32) + (was + low < was ? 1u : 0u);
            if (high) atomicAdd(&s.mass_hi[b[e]], high);
          }
        }
      });
      // The cluster's histogram, two bins a thread.  Each CTA sums its share of
      // the bins, ctas / 2 threads a bin and two CTAs a thread, and writes the
      // sums to all (every CTA reading all bins of all took 3 to 9 us at 16 CTAs).
      uint32_t c[2];
      uint64_t m[2];
      if (p.ctas == 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          c[j] = s.count[2 * tid + j];
          m[j] = s.mass_lo[2 * tid + j] + (static_cast<uint64_t>(s.mass_hi[2 * tid + j]) << 32);
        }
      } else {
        cluster_barrier();
        const int team = p.ctas / 2, bin = static_cast<int>(rank) * (kBins / p.ctas) + tid / team, r0 = tid % team * 2;
        uint32_t sum_c = 0;
        uint64_t sum_m = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Shared *o = at_rank(&s, r0 + j);
          sum_c += o->count[bin];
          if (by_mass) sum_m += o->mass_lo[bin] + (static_cast<uint64_t>(o->mass_hi[bin]) << 32);
        }
        for (int o = 1; o < team; o <<= 1) {
          sum_c += __shfl_xor_sync(0xFFFFFFFFu, sum_c, o);
          sum_m += __shfl_xor_sync(0xFFFFFFFFu, sum_m, o);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Shared *o = at_rank(&s, r0 + j);
          o->sum.count[bin] = sum_c;
          o->sum.mass[bin] = sum_m;
        }
        cluster_barrier();
#pragma unroll
        for (int j = 0; j < 2; ++j) c[j] = s.sum.count[2 * tid + j], m[j] = s.sum.mass[2 * tid + j];
      }
      uint32_t cum_c = c[0] + c[1], all_c;
      uint64_t cum_m = m[0] + m[1], all_m;
      scan(cum_c, cum_m, all_c, all_m, s);
      if (round == 0) {
        if (!by_mass && all_c <= want) return 0;  // no more tokens than that: all stay
        if (by_mass) target = share_of(set.top_p, all_m);
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
      const bool all_of_it = round == 0 && before_count + inside <= kFew;  // the ranges above as well
      if (all_of_it || inside <= kList) {
        // the first round's ranges by their ends: two comparisons instead of the range of every logit
        const float at_bin = 0x1p23f + static_cast<float>(bin), none = -kMinusInf;
        const float from = least_float(hi, [&](float x) { return spot(x) <= at_bin; });
        const float until = all_of_it || bin == 0u || hi == none ? none : least_float(hi, [&](float x) { return spot(x) < at_bin; });
        each4([&](const float (&l)[4], int i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (round == 0) {
              if (!(l[e] >= from && (l[e] < until || until == none))) continue;
            } else if (bin_of(l[e], i + e) != bin) {
              continue;
            }
            if (!among.keeps(l[e], static_cast<int>(begin) + i + e)) continue;
            append(place_of(l[e], begin + static_cast<uint32_t>(i + e)), by_mass && !all_of_it ? weights.of(l[e]) : 0ull);
          }
        });
        const int all = static_cast<int>(listed());
        if (all_of_it) return all;
        if (rank == 0) {
          pull();
          if (tid < all) {
            const uint64_t at = s.pulled[tid], w = s.pulled_w[tid];
            uint32_t c0 = before_count;
            uint64_t m0 = before_mass;
            for (int j = 0; j < all; ++j)
              if (s.pulled[j] < at) ++c0, m0 += s.pulled_w[j];
            if (by_mass ? (m0 < target && target <= m0 + w) : (c0 + 1u == want))
              for (int r = 0; r < p.ctas; ++r) at_rank(&s, r)->place = at;
          }
        }
        if (tid == 0) s.list_n = 0u;
        cluster_barrier();
        cut = Cut{logit_at(s.place), static_cast<int>(index_at(s.place))};
        return 0;
      }
      __syncthreads();  // hit_bin was read
      if (round == 0) range = bin, prefix = 0;
      else prefix = (prefix << 10) | bin;
    }
  };
  uint64_t target = 0;
  int few = 0;
  bool by_count = set.top_k > 0;
  if (by_groups) {
    // The top_k-th largest of the groups' maxima is at most the top_k-th largest
    // logit: what is no less holds the first top_k, and seldom many more.
    // (To 16 bits, found from the top one down by a warp.)
    if (warp == 0) {
      uint32_t key[kGroups / 32], bound = 0u;
#pragma unroll
      for (int e = 0; e < kGroups / 32; ++e) key[e] = ~static_cast<uint32_t>(place_of(s.group[lane + 32 * e], 0) >> kIndexBits);
#pragma unroll 1
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t more = bound | (1u << bit);
        int above = 0;
#pragma unroll
        for (int e = 0; e < kGroups / 32; ++e) above += key[e] >= more;
        if (__reduce_add_sync(0xFFFFFFFFu, above) >= set.top_k) bound = more;
      }
      // fewer groups than that hold a token: not a number
      if (lane == 0) s.bound = __uint_as_float((bound & 0x80000000u) ? bound & 0x7FFFFFFFu : ~bound);
    }
    __syncthreads();
    const float bound = s.bound;
    if (bound > kMinusInf) {
      each4([&](const float (&l)[4], int i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (l[e] >= bound) append(place_of(l[e], begin + static_cast<uint32_t>(i + e)), 0ull);
      });
      const uint32_t all = listed();
      if (all <= kFew) few = static_cast<int>(all);
      else if (tid == 0) s.list_n = 0u;
    }
  }
  if (few == 0 && by_count) few = narrow(false, target);
  if (few == 0 && set.top_p < 1.0f) by_count = false, few = narrow(true, target);
  if (few != 0) {
    if (rank != 0) {
      cluster_barrier();  // rank 0 has read this CTA's list
      return;
    }
    pull();
    cluster_arrive();
    draw_from_list(p, row, set, weights, least, by_count, target, few, s);
    cluster_wait();
    return;
  }

  // ---- the draw: kept weights summed block by block, and walked by index in the block drawn ----
  if (set.min_p > 0.0f) {
    // (The formula's inverse is not near enough where it comes out next to 0.)
    const float l = least_float(hi, [&](float x) { return weights.exponent(x) >= least; });
    if (l > cut.l) cut = Cut{l, kEvery};
  }
  const Cut kept = weighing(cut);
  const int blocks = (n + kBlock - 1) / kBlock;
  for (int b = warp; b < blocks; b += kWarps) {
    uint64_t sum = 0;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int i0 = b * kBlock + part * (kBlock / 2) + lane;
      constexpr int kEach = kBlock / 64;
      float l[kEach];
      uint32_t who[kEach];
      int m = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = i0 + 32 * e;
        l[e] = i < n ? logit<T>(data + i) : kMinusInf;
        who[e] = __ballot_sync(0xFFFFFFFFu, kept.keeps(l[e], static_cast<int>(begin) + i));
        m += __popc(who[e]);
      }
      if (m > kBlock / 4) {  // most are kept
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const bool on = who[e] >> lane & 1u;
          const uint64_t w = weights.of(on ? l[e] : hi);
          sum += on ? w : 0ull;
        }
        continue;
      }
      // else the kept logits side by side, in any order, so that every lane has work
      float *pack = s.pack[warp];
      int at = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (who[e] >> lane & 1u) pack[at + __popc(who[e] & ((1u << lane) - 1u))] = l[e];
        at += __popc(who[e]);
      }
      __syncwarp();
      for (int j = lane; j < m; j += 64) {
        uint64_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) w[e] = weights.of(j + 32 * e < m ? pack[j + 32 * e] : hi);
#pragma unroll
        for (int e = 0; e < 2; ++e) sum += j + 32 * e < m ? w[e] : 0ull;
      }
      __syncwarp();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) s.block_mass[b] = sum;
  }
  __syncthreads();
  const uint64_t mine = tid < blocks ? s.block_mass[tid] : 0ull;
  uint32_t none = 0, none_total;
  uint64_t before = mine, total;
  scan(none, before, none_total, total, s);
  if (tid < p.ctas) at_rank(&s, tid)->rank_mass[rank] = total;
  cluster_barrier();
  uint64_t all = 0, base = 0;
  for (int r = 0; r < p.ctas; ++r) {
    if (r == static_cast<int>(rank)) base = all;
    all += s.rank_mass[r];
  }
  const uint64_t drawn = drawn_at(set.u, all);
  if (drawn < base || drawn >= base + total) return;
  before += base;
  if (before <= drawn && drawn < before + mine) s.hit_bin = static_cast<uint32_t>(tid), s.hit_before_mass = before;
  __syncthreads();
  const int i = static_cast<int>(s.hit_bin) * kBlock + tid;  // a token a thread
  static_assert(kBlock == kThreads, "the block drawn is walked a token a thread");
  const float l = i < n ? logit<T>(data + i) : kMinusInf;
  const bool on = kept.keeps(l, static_cast<int>(begin) + i);
  const uint64_t w = on ? weights.of(l) : 0ull, first = s.hit_before_mass;
  before = w;
  scan(none, before, none_total, total, s);
  before += first;
  if (before <= drawn && drawn < before + w) write_row(p, row, begin + static_cast<uint32_t>(i), l, weights, all);
}

template <typename T>
cudaError_t launch(SampleView p, int rows, int sms, cudaStream_t s) {
  // CTAs of a row: as many as finish soonest, by rounds over the SMs (two CTAs
  // each) times a CTA's tokens and about 8000 tokens' time for its barriers.  Top-p
  // alone, us at 1, 2, 4, 8, 16 CTAs (131072 float32 tokens from 4 on): 296 x 32003
  // bfloat16 54 73 113 203 490 (1 taken); 64 x 32000 36 27 29 45 102 (2); 64 x 131072
  // 80 78 135 (8); 1 x 131072 38 27 22 (16).  It takes one step too many at 16 x 131072
  // (39 35 47: 16 taken), 8 x 32000 (36 25 19 17 23: 16) and 300 x 32003 (84 88: 2).
  constexpr int kMost = 72 * 1024 / sizeof(T);  // tokens that leave room for a second CTA
  constexpr int kMostBytes = 160 * 1024;         // of a CTA's tokens
  constexpr size_t kFirst = (sizeof(Shared) + 15) / 16 * 16 + 16;
  static_assert(kFirst + kMostBytes <= 227 * 1024, "shared memory");
  constexpr int64_t kFixed = 8000;
  int64_t least = INT64_MAX;
  for (int c = 1; c <= kMaxCtas; c *= 2) {
    const int64_t slice = (p.vocab + c - 1) / c;
    if (slice > kMaxBlocks * kBlock || slice * sizeof(T) > kMostBytes) continue;
    const int64_t slots = static_cast<int64_t>(sms) * (slice > kMost ? 1 : 2);
    const int64_t time = (static_cast<int64_t>(rows) * c + slots - 1) / slots * (slice + kFixed);
    if (time < least) least = time, p.ctas = c;
  }
  p.slice = (p.vocab + p.ctas - 1) / p.ctas;
  const size_t smem = kFirst + static_cast<size_t>(p.slice) * sizeof(T);
  static SmemLimit limit;
  cudaError_t e = limit.set(reinterpret_cast<const void *>(k_sample<T>), static_cast<int>(kFirst + kMostBytes));
  if (e == cudaSuccess && p.ctas > 8) e = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  const uint64_t rows64 = a->rows;
  const Span tokens{a->tokens, rows64 * 8}, logprobs{a->logprobs, rows64 * 4};
  const Span inputs[] = {
      {a->logits, ((rows64 - 1) * a->logits_stride + a->vocab) * (a->logits_dtype == FNMOE_DTYPE_F32 ? 4 : 2)},
      {a->uniform, rows64 * 4}, {a->temperatures, rows64 * 4}, {a->top_ks, rows64 * 4}, {a->top_ps, rows64 * 4},
      {a->min_ps, rows64 * 4}};
  bool overlap = tokens.meets(logprobs);
  for (const Span &in : inputs) overlap = overlap || tokens.meets(in) || logprobs.meets(in);
  if (overlap) { err = "tokens and logprobs overlap inputs or one another"; return FNMOE_ERR_VALUE; }
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
