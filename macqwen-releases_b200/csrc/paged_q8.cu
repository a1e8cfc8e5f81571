// paged_q8.cu -- filling and reading the paged 8-bit KV cache on sm_100a:
// block tables and slot maps from request lengths, the quantising append and
// the read-back.  (The attention over it: attention_q8.cu.)
//
// Cache: codes [pages][page_size][Hkv][D] of 8 bits (int8 or e4m3), one
// float32 scale per `block` consecutive tokens of a page and kv head
// [pages][page_size / block][Hkv].  page_size is a multiple of block, so
// slot / block numbers the scale blocks of the whole cache.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "moe_kernels.cuh"
#include "paged_q8.cuh"

namespace fnmoe {

namespace {

// ---- page plan --------------------------------------------------------------
//
// One launch.  Every CTA computes the same prefix sums over the batch into
// shared memory (16 bytes a sequence; B = 512 is two 256-wide scan rounds),
// then takes its share of table rows (a warp per row) and packed tokens (a
// thread per token, its sequence by binary search).  Splitting the sums into
// a kernel of their own would cost a second launch, about as long as this
// whole call; no CTA reads what another one writes, so none waits.
//
// Bytes: the table read and written once (8 B a cell), 16 B a token, the
// lengths once per CTA (from L2).  Measured: 8.3 us for 16 rows of 512 columns,
// 8.4 us for 512 rows of 256 columns and 26,000 tokens; a chain of latencies:
// lengths, sums, and up to `width` / 32 rounds of load and store over the columns,
// which stay in order since the table may be updated in place.  Below the 11 us
// that a call costs the host.

constexpr int kPlanThreads = 256;
constexpr int kPlanMaxBatch = 8192;

struct PlanView {
  const int32_t *seq_lens, *new_lens, *release, *table;
  int32_t *ring;
  const int32_t *state;
  int32_t *table_out, *lens_out, *state_out;
  int64_t *slot_map;
  int32_t *token_seq, *positions, *cu_new, *admitted;
  int B, page, width, num, cap;
};

struct Sum3 {
  long long a, b, c;
};

// Inclusive sums over the block's threads in thread order, plus `carry`
// (which becomes the block's total).  red: 3 * 8 slots of shared memory.
__device__ __forceinline__ Sum3 block_scan(Sum3 v, Sum3 &carry, long long *red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long a = __shfl_up_sync(0xFFFFFFFFu, v.a, off);
    const long long b = __shfl_up_sync(0xFFFFFFFFu, v.b, off);
    const long long c = __shfl_up_sync(0xFFFFFFFFu, v.c, off);
    if (lane >= off) {
      v.a += a;
      v.b += b;
      v.c += c;
    }
  }
  constexpr int W = kPlanThreads / 32;
  __syncthreads();  // red may still be read by the previous round
  if (lane == 31) {
    red[warp] = v.a;
    red[W + warp] = v.b;
    red[2 * W + warp] = v.c;
  }
  __syncthreads();
  Sum3 before = carry;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const long long a = red[w], b = red[W + w], c = red[2 * W + w];
    if (w < warp) {
      before.a += a;
      before.b += b;
      before.c += c;
    }
    carry.a += a;
    carry.b += b;
    carry.c += c;
  }
  v.a += before.a;
  v.b += before.b;
  v.c += before.c;
  return v;
}

// Pages of `tokens` tokens; both are ints, their sum may not be one.
__device__ __forceinline__ int pages_of(int tokens, int page) {
  return static_cast<int>((static_cast<uint32_t>(tokens) + static_cast<uint32_t>(page) - 1u) / static_cast<uint32_t>(page));
}

__global__ void __launch_bounds__(kPlanThreads) k_page_plan(PlanView p) {
  extern __shared__ int32_t plan_sm[];
  __shared__ long long red[3 * (kPlanThreads / 32)];
  const int B = p.B, tid = threadIdx.x;
  int32_t *s_held = plan_sm;       // [B] tokens before the new ones
  int32_t *s_start = s_held + B;   // [B] index of the sequence's first new page among those given
  int32_t *s_back = s_start + B;   // [B + 1] pages released before the sequence
  int32_t *s_cu = s_back + B + 1;  // [B + 1] packed tokens before the sequence
  const long long num = p.num;
  const long long head = static_cast<uint32_t>(p.state[0]) % static_cast<uint32_t>(p.num);
  const long long count = min(max(p.state[1], 0), p.num);
  const int row_cap_pages = p.width;

  // Sums of pages wanted, tokens wanted and pages released, and from them
  // which sequences are admitted; then the packed offsets of those.
  Sum3 carry = {0, 0, 0}, carry_n = {0, 0, 0};
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    Sum3 v = {0, 0, 0};
    long long held = 0, n = 0;
    bool fits = false;
    if (b < B) {
      const long long had = max(p.seq_lens[b], 0);
      const bool gone = p.release != nullptr && p.release[b] != 0;
      held = gone ? 0 : had;
      n = max(p.new_lens[b], 0);
      fits = held + n <= static_cast<long long>(row_cap_pages) * p.page;
      if (fits) {
        v.a = (held + n + p.page - 1) / p.page - (held + p.page - 1) / p.page;
        v.b = n;
      }
      if (gone) v.c = min((had + p.page - 1) / p.page, static_cast<long long>(row_cap_pages));
    }
    const Sum3 s = block_scan(v, carry, red);
    const bool ok = fits && (v.a == 0 || s.a <= count) && (v.b == 0 || s.b <= p.cap);
    Sum3 w = {ok ? n : 0, ok ? v.a : 0, 0};
    const Sum3 t = block_scan(w, carry_n, red);
    if (b < B) {
      s_held[b] = static_cast<int32_t>(held);
      s_start[b] = static_cast<int32_t>(t.b - w.b);
      s_back[b] = static_cast<int32_t>(s.c - v.c);
      s_cu[b] = static_cast<int32_t>(t.a - w.a);
      if (blockIdx.x == 0) {
        p.lens_out[b] = static_cast<int32_t>(held + w.a);
        p.admitted[b] = ok ? 1 : 0;
        p.cu_new[b] = s_cu[b];
      }
    }
  }
  if (tid == 0) {
    s_back[B] = static_cast<int32_t>(carry.c);
    s_cu[B] = static_cast<int32_t>(carry_n.a);
    if (blockIdx.x == 0) {
      p.cu_new[B] = s_cu[B];
      p.state_out[0] = static_cast<int32_t>((head + carry_n.b) % num);
      p.state_out[1] = static_cast<int32_t>(min(count - carry_n.b + carry.c, num));
    }
  }
  __syncthreads();

  // Table rows.  A released row's pages go to the ring's end before its cells
  // are overwritten (by the same thread: the table may be updated in place).
  const int gwarp = blockIdx.x * (kPlanThreads / 32) + (tid >> 5), warps = gridDim.x * (kPlanThreads / 32);
  for (int b = gwarp; b < B; b += warps) {
    const int held = s_held[b], n = s_cu[b + 1] - s_cu[b];
    const int pages0 = pages_of(held, p.page), pages1 = pages_of(held + n, p.page);
    const int back0 = s_back[b], back = s_back[b + 1] - back0;
    const bool gone = p.release != nullptr && p.release[b] != 0;
    const size_t row = static_cast<size_t>(b) * p.width;
    const int start = s_start[b];
    for (int c = tid & 31; c < p.width; c += 32) {
      const int32_t old = p.table[row + c];
      if (c < back) p.ring[(head + count + back0 + c) % num] = old;
      int32_t now = gone ? -1 : old;
      if (c >= pages0 && c < pages1) now = p.ring[(head + start + (c - pages0)) % num];
      p.table_out[row + c] = now;
    }
  }

  // Packed tokens: slot, sequence and position.  Their pages come from the
  // input table (held pages; never cleared, since a released row holds none)
  // or the ring, not from the output table, which other CTAs are writing.
  const int total = s_cu[B];
  for (int t = blockIdx.x * kPlanThreads + tid; t < p.cap; t += gridDim.x * kPlanThreads) {
    long long slot = -1;
    int seq = -1, pos = -1;
    if (t < total) {
      int lo = 0, hi = B;  // the last sequence that starts at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      seq = lo;
      pos = s_held[seq] + t - s_cu[seq];
      const int c = pos / p.page;
      const int pages0 = pages_of(s_held[seq], p.page);
      const int page = c < pages0 ? p.table[static_cast<size_t>(seq) * p.width + c]
                                  : p.ring[(head + s_start[seq] + (c - pages0)) % num];
      slot = page < 0 ? -1 : static_cast<long long>(page) * p.page + (pos - c * p.page);
    }
    p.slot_map[t] = slot;
    p.token_seq[t] = seq;
    p.positions[t] = pos;
  }
}

// ---- quantising append ------------------------------------------------------
//
// A run is the rows of one scale block that the call writes (adjacent in the
// map, ascending slots).  One CTA takes a run's rows of one kv head, of K or
// of V, whole: 16-byte loads into registers (at most 64 a thread), the
// largest magnitude over the CTA as an integer maximum of the bf16 bits, then
// the codes.  The rows are so read once and written once; the codes already
// in the block are read only when the block's scale grows.
//
// Grid: chunks of `chunk` tokens x (kv head, K or V); a CTA handles the runs
// that begin in its chunk.  The host picks the chunk from the token count so
// that a decode batch gets a CTA per row and a prefill chunk does not launch
// a CTA per token.  Measured: 5,000 rows of 2 heads of 256, 12.5 us (15 MB;
// 2.4 us at HBM rate): a CTA's chain of slots, rows, maximum and codes.

constexpr int kAppendThreads = 256;
constexpr int kMaxBlock = 128;
constexpr float kQ8Tiny = 0x1p-100f;  // least magnitude a scale is made for

struct Q8Store {
  const uint16_t *x[2];
  uint64_t stride[2];
  uint8_t *codes[2];
  float *scale[2];
  const int64_t *slots;
  int64_t n_slots;  // of the cache
  int tokens, chunk, block, block_shift, Hkv;
};

template <bool E4M3>
struct Q8Code;

template <>
struct Q8Code<false> {
  static constexpr float kTop = 127.0f;
  // Four codes (one word) to float.
  static __device__ __forceinline__ void decode4(uint32_t w, float f[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xFFu));
  }
  // Four finite floats within +-kTop to codes, nearest even.
  static __device__ __forceinline__ uint32_t encode4(const float f[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (static_cast<uint32_t>(__float2int_rn(f[i])) & 0xFFu) << (8 * i);
    return w;
  }
};

template <>
struct Q8Code<true> {
  static constexpr float kTop = 448.0f;
  static __device__ __forceinline__ void decode4(uint32_t w, float f[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h;
      asm("{\n .reg .b16 lo;\n mov.b16 lo, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}\n"
          : "=r"(h)
          : "h"(static_cast<uint16_t>(w >> (16 * i))));
      const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint32_t encode4(const float f[4]) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(f[1]), "f"(f[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(f[3]), "f"(f[2]));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
};

__device__ __forceinline__ float clamp_top(float v, float top) { return fminf(fmaxf(v, -top), top); }

// Eight bf16 (one uint4) times inv to eight codes; NaN becomes 0.
template <bool E4M3>
__device__ __forceinline__ uint2 encode_row8(uint4 v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = bf16_to_f32(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
    f[i] = x != x ? 0.0f : clamp_top(__fmul_rn(x, inv), Q8Code<E4M3>::kTop);
  }
  return make_uint2(Q8Code<E4M3>::encode4(f), Q8Code<E4M3>::encode4(f + 4));
}

// Largest finite bf16 magnitude of eight values, as its bits.
__device__ __forceinline__ uint32_t peak8(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = (w[i >> 1] >> (16 * (i & 1))) & 0x7FFFu;
    m = max(m, b < 0x7F80u ? b : 0u);
  }
  return m;
}

// The codes of rows row0, row0 + step, ... below `rows` (eight each, at `a`,
// `pitch` bytes from row to row) rounded again to a scale 1 / shrink times as large.
template <int D, bool E4M3>
__device__ __forceinline__ void requantise(uint8_t *a, uint64_t pitch, int row0, int step, int rows, float shrink) {
  for (int r = row0; r < rows; r += step) {
    uint2 *at = reinterpret_cast<uint2 *>(a + static_cast<uint64_t>(r) * pitch);
    const uint2 q = *at;
    float f[8];
    Q8Code<E4M3>::decode4(q.x, f);
    Q8Code<E4M3>::decode4(q.y, f + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e)  // a slot that was never written may hold a NaN code
      f[e] = f[e] != f[e] ? 0.0f : clamp_top(__fmul_rn(f[e], shrink), Q8Code<E4M3>::kTop);
    *at = make_uint2(Q8Code<E4M3>::encode4(f), Q8Code<E4M3>::encode4(f + 4));
  }
}

// D: head dim; NP: passes of the CTA over a block's rows.
template <int D, int NP, bool E4M3>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append_q8(Q8Store p) {
  constexpr int kTpr = D / 8;                        // threads per row, 8 values each
  constexpr int kRows = kAppendThreads / kTpr;       // rows per pass
  constexpr float kTop = Q8Code<E4M3>::kTop;
  __shared__ int64_t s_slot[1 + 2 * kMaxBlock];      // slots of tokens t0 - 1 .. t0 + chunk + block
  __shared__ uint32_t s_peak[kAppendThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int side = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int t0 = blockIdx.x * p.chunk;
  const int t1 = min(p.tokens, t0 + p.chunk);
  for (int i = tid; i < 1 + p.chunk + p.block; i += kAppendThreads) {
    const int t = t0 - 1 + i;
    s_slot[i] = t >= 0 && t < p.tokens ? p.slots[t] : -1;
  }
  __syncthreads();
  const uint16_t *x = p.x[side];
  const uint64_t stride = p.stride[side];
  uint8_t *codes = p.codes[side];
  float *scales = p.scale[side];
  const int row = tid / kTpr, col = (tid % kTpr) * 8;
  const uint32_t bmask = static_cast<uint32_t>(p.block - 1);

  for (int c0 = t0; c0 < t1; c0 += 32) {
    // Runs begin at slots that do not continue the token before.
    const int tl = c0 + lane;
    bool begins = false;
    if (tl < t1) {
      const int64_t s = s_slot[tl - t0 + 1], before = s_slot[tl - t0];
      begins = s >= 0 && s < p.n_slots &&
               !((static_cast<uint32_t>(s) & bmask) != 0 && before >= 0 && before == s - 1);
    }
    uint32_t runs = __ballot_sync(0xFFFFFFFFu, begins);
    while (runs) {
      const int t = c0 + __ffs(runs) - 1;
      runs &= runs - 1;
      const int64_t slot = s_slot[t - t0 + 1];
      const int first = static_cast<int>(static_cast<uint32_t>(slot) & bmask);
      const int64_t block = slot >> p.block_shift;
      int len = 0;  // rows of the run
      const int most = p.block - first;
      for (int j0 = 0; j0 < most; j0 += 32) {
        const int j = j0 + lane;
        const bool in = j < most && t + j < p.tokens && s_slot[t - t0 + 1 + j] == slot + j;
        const uint32_t m = __ballot_sync(0xFFFFFFFFu, in);
        if (m != 0xFFFFFFFFu) {
          len = j0 + __ffs(~m) - 1;
          break;
        }
        len = j0 + 32;
      }
      float *sp = scales + block * p.Hkv + h;
      const float old = first > 0 ? *sp : 0.0f;
      uint4 v[NP];
      uint32_t peak = 0;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * kRows + row;
        v[i] = make_uint4(0, 0, 0, 0);
        if (r < len)
          v[i] = __ldg(reinterpret_cast<const uint4 *>(x + static_cast<uint64_t>(t + r) * stride +
                                                       static_cast<uint64_t>(h) * D + col));
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) peak = max(peak, peak8(v[i]));
      peak = __reduce_max_sync(0xFFFFFFFFu, peak);
      __syncthreads();  // s_peak may still be read for the run before
      if (lane == 0) s_peak[warp] = peak;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) peak = max(peak, s_peak[w]);
      const float mag = fmaxf(bf16_to_f32(static_cast<uint16_t>(peak)), kQ8Tiny);
      const float scale = fmaxf(old, __fdiv_rn(mag, kTop));
      const float inv = __fdiv_rn(1.0f, scale);
      const int64_t slot0 = slot - first;
      auto at = [&](int r) {  // 8 codes of the block's row r
        return reinterpret_cast<uint2 *>(codes + (static_cast<uint64_t>(slot0 + r) * p.Hkv + h) * D + col);
      };
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * kRows + row;
        if (r < len) *at(first + r) = encode_row8<E4M3>(v[i], inv);
      }
      if (first > 0 && scale != old) {
        requantise<D, E4M3>(codes + (static_cast<uint64_t>(slot0) * p.Hkv + h) * D + col, static_cast<uint64_t>(p.Hkv) * D, row,
                            kRows, first, __fdiv_rn(old, scale));
      }
      if (tid == 0) *sp = scale;  // every thread has read the old one (two barriers ago)
    }
  }
}

// Small blocks (at most 4,096 values a head): a warp takes a run's rows of one
// kv head, of K or of V, so that neither a barrier nor shared memory stands
// between its loads, its maximum and its stores; the CTA's warps take
// different heads.  With a CTA a run, 13,000 rows of 8 heads of 128 in blocks
// of 16 took 53 us; this takes 36 us (10,500 rows: 29 us, 65 MB).
template <int D, int NP, bool E4M3>
__global__ void __launch_bounds__(256) k_kv_append_q8_small(Q8Store p) {
  constexpr int kTpr = D / 8, kRows = 32 / kTpr;  // lanes per row, rows per pass
  constexpr float kTop = Q8Code<E4M3>::kTop;
  __shared__ int64_t s_slot[1 + 2 * kMaxBlock];
  const int lane = threadIdx.x & 31, item = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int t0 = blockIdx.x * p.chunk, t1 = min(p.tokens, t0 + p.chunk);
  for (int i = threadIdx.x; i < 1 + p.chunk + p.block; i += blockDim.x) {
    const int t = t0 - 1 + i;
    s_slot[i] = t >= 0 && t < p.tokens ? p.slots[t] : -1;
  }
  __syncthreads();
  if (item >= 2 * p.Hkv) return;
  const int side = item & 1, h = item >> 1;
  const uint16_t *x = p.x[side];
  const uint64_t stride = p.stride[side];
  float *scales = p.scale[side];
  const int row = lane / kTpr, col = (lane % kTpr) * 8;
  const uint32_t bmask = static_cast<uint32_t>(p.block - 1);
  for (int c0 = t0; c0 < t1; c0 += 32) {
    const int tl = c0 + lane;
    bool begins = false;
    if (tl < t1) {
      const int64_t s = s_slot[tl - t0 + 1], before = s_slot[tl - t0];
      begins = s >= 0 && s < p.n_slots &&
               !((static_cast<uint32_t>(s) & bmask) != 0 && before >= 0 && before == s - 1);
    }
    uint32_t runs = __ballot_sync(0xFFFFFFFFu, begins);
    while (runs) {
      const int t = c0 + __ffs(runs) - 1;
      runs &= runs - 1;
      const int64_t slot = s_slot[t - t0 + 1];
      const int first = static_cast<int>(static_cast<uint32_t>(slot) & bmask);
      float *sp = scales + (slot >> p.block_shift) * p.Hkv + h;
      const float old = first > 0 ? *sp : 0.0f;
      const int most = min(p.block - first, p.tokens - t);
      const uint16_t *src = x + static_cast<uint64_t>(t) * stride + static_cast<uint64_t>(h) * D + col;
      uint4 v[NP];
      uint32_t peak = 0, here = 0;  // bit i: pass i's row is of the run
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * kRows + row;
        v[i] = make_uint4(0, 0, 0, 0);
        if (r < most && s_slot[t - t0 + 1 + r] == slot + r) {  // slots ascend: a run has no gap
          here |= 1u << i;
          v[i] = __ldg(reinterpret_cast<const uint4 *>(src + static_cast<uint64_t>(r) * stride));
        }
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) peak = max(peak, peak8(v[i]));
      peak = __reduce_max_sync(0xFFFFFFFFu, peak);
      const float mag = fmaxf(bf16_to_f32(static_cast<uint16_t>(peak)), kQ8Tiny);
      const float scale = fmaxf(old, __fdiv_rn(mag, kTop));
      const float inv = __fdiv_rn(1.0f, scale);
      uint8_t *dst = p.codes[side] + (static_cast<uint64_t>(slot - first) * p.Hkv + h) * D + col;
      const uint64_t pitch = static_cast<uint64_t>(p.Hkv) * D;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if ((here >> i) & 1u)
          *reinterpret_cast<uint2 *>(dst + static_cast<uint64_t>(first + i * kRows + row) * pitch) = encode_row8<E4M3>(v[i], inv);
      if (first > 0 && scale != old) requantise<D, E4M3>(dst, pitch, row, kRows, first, __fdiv_rn(old, scale));
      __syncwarp();  // every lane has read the old scale
      if (lane == 0) *sp = scale;
    }
  }
}

// ---- read-back --------------------------------------------------------------
//
// A thread takes 16 codes of K and the same 16 of V of one slot: two 16-byte
// loads, four 16-byte stores.  3 bytes a value moved.  32,768 slots of 2 heads
// of 256: 23 us, 4.4 TB/s, two thirds of HBM (8 codes a thread 25 us, two or four
// such pieces a thread 23 and 25 us).

struct Q8Load {
  const uint8_t *codes[2];
  const float *scale[2];
  uint16_t *out[2];
  const int64_t *slots;
  int64_t n_slots;
  uint64_t items;
  uint32_t units, block_shift, Hkv, d_shift;  // units: 16-code pieces of a slot's row
};

template <bool E4M3>
__device__ __forceinline__ void widen16(uint4 q, float s, uint4 o[2]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
    Q8Code<E4M3>::decode4(w[i], f);
#pragma unroll
    for (int e = 0; e < 4; e += 2)
      r[2 * i + e / 2] = static_cast<uint32_t>(f32_to_bf16(__fmul_rn(f[e], s))) |
                         (static_cast<uint32_t>(f32_to_bf16(__fmul_rn(f[e + 1], s))) << 16);
  }
  o[0] = make_uint4(r[0], r[1], r[2], r[3]);
  o[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

template <bool E4M3>
__global__ void __launch_bounds__(256) k_kv_read_q8(Q8Load p) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.items) return;
  const uint64_t n = i / p.units;
  const uint32_t u = static_cast<uint32_t>(i - n * p.units);
  const int64_t slot = p.slots[n];
  uint4 o[2][2] = {};
  if (slot >= 0 && slot < p.n_slots) {
    const uint64_t at = static_cast<uint64_t>(slot) * p.units + u;
    const uint64_t sc = (static_cast<uint64_t>(slot) >> p.block_shift) * p.Hkv + ((u * 16) >> p.d_shift);
    const uint4 q0 = __ldg(reinterpret_cast<const uint4 *>(p.codes[0]) + at);
    const uint4 q1 = __ldg(reinterpret_cast<const uint4 *>(p.codes[1]) + at);
    const float s0 = __ldg(p.scale[0] + sc), s1 = __ldg(p.scale[1] + sc);
    widen16<E4M3>(q0, s0, o[0]);
    widen16<E4M3>(q1, s1, o[1]);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint4 *dst = reinterpret_cast<uint4 *>(p.out[x]) + 2 * i;
    dst[0] = o[x][0];
    dst[1] = o[x][1];
  }
}

template <int D, int NP>
void launch_append(const Q8Store &p, dim3 grid, bool e4m3, cudaStream_t s) {
  if (e4m3)
    k_kv_append_q8<D, NP, true><<<grid, kAppendThreads, 0, s>>>(p);
  else
    k_kv_append_q8<D, NP, false><<<grid, kAppendThreads, 0, s>>>(p);
}

template <int D, int NP>
void launch_append_small(const Q8Store &p, dim3 grid, int warps, bool e4m3, cudaStream_t s) {
  if (e4m3)
    k_kv_append_q8_small<D, NP, true><<<grid, 32 * warps, 0, s>>>(p);
  else
    k_kv_append_q8_small<D, NP, false><<<grid, 32 * warps, 0, s>>>(p);
}

template <int D>
void launch_append_d(Q8Store p, bool e4m3, cudaStream_t s) {
  const int items = 2 * p.Hkv, values = p.block * D;
  const bool small = values <= 4096;
  const int warps = std::min(items, 8);
  const unsigned across = small ? (items + warps - 1) / warps : items;
  // Chunks of one token while that gives every SM four CTAs, of a block at most.
  const uint64_t ctas = static_cast<uint64_t>(p.tokens) * across / (148 * 4);
  p.chunk = static_cast<int>(std::min<uint64_t>(std::max<uint64_t>(ctas, 1), p.block));
  const dim3 grid((p.tokens + p.chunk - 1) / p.chunk, across);
  if (small) {
    if constexpr (D == 64) {
      if (p.block == 16) return launch_append_small<D, 4>(p, grid, warps, e4m3, s);
    }
    if constexpr (D <= 128) {
      if (values == 2048) return launch_append_small<D, 8>(p, grid, warps, e4m3, s);
    }
    return launch_append_small<D, 16>(p, grid, warps, e4m3, s);
  }
  constexpr int kRows = kAppendThreads / (D / 8);
  const int np = (p.block + kRows - 1) / kRows;
  if (np <= 4) return launch_append<D, 4>(p, grid, e4m3, s);
  if constexpr (D >= 128) {
    if (np <= 8) return launch_append<D, 8>(p, grid, e4m3, s);
  }
  if constexpr (D >= 256) return launch_append<D, 16>(p, grid, e4m3, s);
}

int launched(const char *what, std::string &err) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return FNMOE_OK;
  err = std::string(what) + ": " + cudaGetErrorString(e);
  return FNMOE_ERR_LAUNCH;
}

int shift_of(uint32_t power) { return 31 - __builtin_clz(power); }

bool misaligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace

int check_q8_cache(const FnQ8Cache &c, std::string &err) {
  if (!c.k_codes || !c.v_codes || !c.k_scale || !c.v_scale) {
    err = "k_codes, v_codes, k_scale and v_scale are required";
    return FNMOE_ERR_NULL;
  }
  if (c.code_type != FNMOE_Q8_INT8 && c.code_type != FNMOE_Q8_E4M3) {
    err = "code_type must be FNMOE_Q8_INT8 or FNMOE_Q8_E4M3";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (c.block != 16 && c.block != 32 && c.block != 64 && c.block != 128) {
    err = "block must be 16, 32, 64 or 128 tokens";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) {
    err = "head_dim must be 64, 128 or 256";
    return FNMOE_ERR_UNSUPPORTED;
  }
  if (c.num_pages == 0 || c.num_pages > 0x7FFFFFFFu || c.page_size == 0 || c.page_size > (1u << 20) ||
      c.page_size % c.block || c.kv_heads == 0 || c.kv_heads > 32767u ||
      static_cast<uint64_t>(c.num_pages) * c.page_size > 0x7FFFFFFFull) {
    err = "the cache needs pages, kv heads, a page_size that is a multiple of block and fewer than 2^31 slots";
    return FNMOE_ERR_SHAPE;
  }
  if (misaligned(c.k_codes, 16) || misaligned(c.v_codes, 16) || misaligned(c.k_scale, 4) ||
      misaligned(c.v_scale, 4)) {
    err = "k_codes and v_codes must be 16-byte and the scales 4-byte aligned";
    return FNMOE_ERR_VALUE;
  }
  return FNMOE_OK;
}

int page_plan(const FnPagePlanArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (!a->seq_lens || !a->new_lens || !a->block_table || !a->free_pages || !a->free_state || !a->block_table_out ||
      !a->seq_lens_out || !a->free_state_out || !a->slot_map || !a->token_seq || !a->positions || !a->cu_new ||
      !a->admitted) {
    err = "every array but release is required";
    return FNMOE_ERR_NULL;
  }
  if (a->batch == 0 || a->page_size == 0 || a->max_pages == 0 || a->num_pages == 0 || a->max_tokens == 0 ||
      a->num_pages > 0x7FFFFFFFu || a->max_tokens > 0x7FFFFFFFu ||
      static_cast<uint64_t>(a->max_pages) * a->page_size > 0x7FFFFFFFull) {
    err = "batch, page_size, max_pages, num_pages and max_tokens must be positive and a table row's tokens below 2^31";
    return FNMOE_ERR_SHAPE;
  }
  if (a->batch > kPlanMaxBatch) {
    err = "at most " + std::to_string(kPlanMaxBatch) + " sequences";
    return FNMOE_ERR_SHAPE;
  }
  for (const void *at : {static_cast<const void *>(a->seq_lens), static_cast<const void *>(a->new_lens),
                         static_cast<const void *>(a->release), static_cast<const void *>(a->block_table),
                         static_cast<const void *>(a->free_pages), static_cast<const void *>(a->free_state),
                         static_cast<const void *>(a->block_table_out), static_cast<const void *>(a->seq_lens_out),
                         static_cast<const void *>(a->free_state_out), static_cast<const void *>(a->token_seq),
                         static_cast<const void *>(a->positions), static_cast<const void *>(a->cu_new),
                         static_cast<const void *>(a->admitted)}) {
    if (misaligned(at, 4)) { err = "the int32 arrays must be 4-byte aligned"; return FNMOE_ERR_VALUE; }
  }
  if (misaligned(a->slot_map, 8)) { err = "slot_map must be 8-byte aligned"; return FNMOE_ERR_VALUE; }
  if (a->seq_lens_out == a->seq_lens || a->free_state_out == a->free_state) {
    err = "seq_lens_out and free_state_out must not be the inputs (other CTAs still read those)";
    return FNMOE_ERR_VALUE;
  }
  PlanView p{};
  p.seq_lens = a->seq_lens;
  p.new_lens = a->new_lens;
  p.release = a->release;
  p.table = a->block_table;
  p.ring = a->free_pages;
  p.state = a->free_state;
  p.table_out = a->block_table_out;
  p.lens_out = a->seq_lens_out;
  p.state_out = a->free_state_out;
  p.slot_map = a->slot_map;
  p.token_seq = a->token_seq;
  p.positions = a->positions;
  p.cu_new = a->cu_new;
  p.admitted = a->admitted;
  p.B = static_cast<int>(a->batch);
  p.page = static_cast<int>(a->page_size);
  p.width = static_cast<int>(a->max_pages);
  p.num = static_cast<int>(a->num_pages);
  p.cap = static_cast<int>(a->max_tokens);
  const size_t smem = sizeof(int32_t) * (4 * static_cast<size_t>(p.B) + 2);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k_page_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) { err = std::string("page plan: ") + cudaGetErrorString(e); return FNMOE_ERR_LAUNCH; }
  }
  // A warp per table row and a thread per token, at most one CTA per SM.
  const uint64_t rows = (a->batch + kPlanThreads / 32 - 1) / (kPlanThreads / 32);
  const uint64_t toks = (static_cast<uint64_t>(a->max_tokens) + kPlanThreads - 1) / kPlanThreads;
  const unsigned grid = static_cast<unsigned>(std::min<uint64_t>(std::max(rows, toks), 148));
  k_page_plan<<<grid, kPlanThreads, smem, s>>>(p);
  return launched("page plan", err);
}

int kv_append_q8(const FnQ8AppendArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (const int rc = check_q8_cache(a->cache, err)) return rc;
  if (a->tokens == 0) return FNMOE_OK;
  if (!a->k || !a->v || !a->slot_map) { err = "k, v and slot_map are required"; return FNMOE_ERR_NULL; }
  const FnQ8Cache &c = a->cache;
  const uint64_t row = static_cast<uint64_t>(c.kv_heads) * c.head_dim;
  if (a->tokens > 0x7FFFFFFFu || a->k_stride < row || a->v_stride < row) {
    err = "token strides must cover a row of kv_heads * head_dim values";
    return FNMOE_ERR_SHAPE;
  }
  if (misaligned(a->k, 16) || misaligned(a->v, 16) || a->k_stride % 8 || a->v_stride % 8 ||
      misaligned(a->slot_map, 8)) {
    err = "k and v must be 16-byte aligned with token strides that are multiples of 8 values, slot_map 8-byte aligned";
    return FNMOE_ERR_VALUE;
  }
  Q8Store p{};
  p.x[0] = static_cast<const uint16_t *>(a->k);
  p.x[1] = static_cast<const uint16_t *>(a->v);
  p.stride[0] = a->k_stride;
  p.stride[1] = a->v_stride;
  p.codes[0] = static_cast<uint8_t *>(c.k_codes);
  p.codes[1] = static_cast<uint8_t *>(c.v_codes);
  p.scale[0] = c.k_scale;
  p.scale[1] = c.v_scale;
  p.slots = a->slot_map;
  p.n_slots = static_cast<int64_t>(c.num_pages) * c.page_size;
  p.tokens = static_cast<int>(a->tokens);
  p.block = static_cast<int>(c.block);
  p.block_shift = shift_of(c.block);
  p.Hkv = static_cast<int>(c.kv_heads);
  const bool e4m3 = c.code_type == FNMOE_Q8_E4M3;
  switch (c.head_dim) {
    case 64: launch_append_d<64>(p, e4m3, s); break;
    case 128: launch_append_d<128>(p, e4m3, s); break;
    default: launch_append_d<256>(p, e4m3, s); break;
  }
  return launched("kv append", err);
}

int kv_read_q8(const FnQ8ReadArgs *a, cudaStream_t s, std::string &err) {
  if (a == nullptr) { err = "args is NULL"; return FNMOE_ERR_NULL; }
  if (a->abi_version != FNMOE_ABI_VERSION) { err = "abi_version mismatch"; return FNMOE_ERR_ABI; }
  if (const int rc = check_q8_cache(a->cache, err)) return rc;
  if (a->count == 0) return FNMOE_OK;
  if (!a->slots || !a->k_out || !a->v_out) { err = "slots, k_out and v_out are required"; return FNMOE_ERR_NULL; }
  if (misaligned(a->k_out, 16) || misaligned(a->v_out, 16) || misaligned(a->slots, 8)) {
    err = "k_out and v_out must be 16-byte and slots 8-byte aligned";
    return FNMOE_ERR_VALUE;
  }
  const FnQ8Cache &c = a->cache;
  Q8Load p{};
  p.codes[0] = static_cast<const uint8_t *>(c.k_codes);
  p.codes[1] = static_cast<const uint8_t *>(c.v_codes);
  p.scale[0] = c.k_scale;
  p.scale[1] = c.v_scale;
  p.out[0] = static_cast<uint16_t *>(a->k_out);
  p.out[1] = static_cast<uint16_t *>(a->v_out);
  p.slots = a->slots;
  p.n_slots = static_cast<int64_t>(c.num_pages) * c.page_size;
  p.units = c.kv_heads * c.head_dim / 16;
  p.items = static_cast<uint64_t>(a->count) * p.units;
  p.block_shift = shift_of(c.block);
  p.Hkv = c.kv_heads;
  p.d_shift = shift_of(c.head_dim);
  const uint64_t blocks = (p.items + 255) / 256;
  if (blocks > 0x7FFFFFFFull) { err = "too many slots"; return FNMOE_ERR_SHAPE; }
  if (c.code_type == FNMOE_Q8_E4M3)
    k_kv_read_q8<true><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
  else
    k_kv_read_q8<false><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
  return launched("kv read", err);
}

}  // namespace fnmoe
