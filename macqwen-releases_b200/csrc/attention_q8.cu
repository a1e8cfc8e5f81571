// attention_q8.cu -- causal attention over the paged 8-bit KV cache (sm_100a).
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale * q_i . k_j - m_i),
//   k_j = ks[block of j] * kcode_j,  v_j = vs[block of j] * vcode_j,
//   j over the positions up to row i's own whose page is in the cache.
//
// Simplest form: one CTA per (row, query head); each warp takes every fourth
// token, a lane D / 32 dims of it.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cmath>
#include <string>

#include "common.cuh"
#include "moe_kernels.cuh"
#include "paged_q8.cuh"

namespace fnmoe {

namespace {

struct Q8View {
  const uint16_t *q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *ctx, *cu;
  uint16_t *out;
  uint64_t q_stride;
  int B, rows, Hq, Hkv, gq, page, block, width, pages;
  float scale;
};

template <bool E4M3>
__device__ __forceinline__ float code_value(uint8_t c) {
  if (!E4M3) return static_cast<float>(static_cast<int8_t>(c));
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(static_cast<uint16_t>(c)));
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(128) k_q8_attention(Q8View p) {
  constexpr int N = D / 32;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  const int r = blockIdx.x / p.Hq, head = blockIdx.x - r * p.Hq, h = head / p.gq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b = r, last;
  if (p.cu) {
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid] <= r) lo = mid; else hi = mid;
    }
    b = lo;
    if (r < p.cu[b] || r >= p.cu[b + 1]) return;
    last = p.ctx[b] - p.cu[b + 1] + r;
  } else {
    last = p.ctx[b] - 1;
  }
  const int seen = min(last + 1, p.width * p.page);
  float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = bf16_to_f32(p.q[static_cast<uint64_t>(r) * p.q_stride + static_cast<uint64_t>(head) * D + i * 32 + lane]) *
           p.scale;
    o[i] = 0.0f;
  }
  for (int t = warp; t < seen; t += 4) {
    const int c = t / p.page;
    const int pg = p.table[static_cast<size_t>(b) * p.width + c];
    if (pg < 0 || pg >= p.pages) continue;
    const size_t slot = static_cast<size_t>(pg) * p.page + (t - c * p.page);
    const size_t at = (slot * p.Hkv + h) * D + lane, sc = slot / p.block * p.Hkv + h;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += q[i] * code_value<E4M3>(p.kc[at + 32 * i]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
    s *= p.ks[sc];
    const float mn = fmaxf(m, s), al = expf(m - mn), w = expf(s - mn);
    m = mn;
    l = l * al + w;
    const float wv = w * p.vs[sc];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * al + wv * code_value<E4M3>(p.vc[at + 32 * i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s_o[warp][32 * i + lane] = o[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  const float mm = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float w[4], L = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = s_m[i] == -INFINITY ? 0.0f : expf(s_m[i] - mm);
    L += w[i] * s_l[i];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v += w[i] * s_o[i][d];
    p.out[(static_cast<size_t>(r) * p.Hq + head) * D + d] = f32_to_bf16(L > 0.0f ? v / L : 0.0f);
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

constexpr uint64_t kWorkspaceBytes = 256;  // nothing kept there yet

template <int D>
void launch(const Q8View &p, bool e4m3, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.rows) * p.Hq;
  if (e4m3)
    k_q8_attention<D, true><<<grid, 128, 0, s>>>(p);
  else
    k_q8_attention<D, false><<<grid, 128, 0, s>>>(p);
}

}  // namespace

int paged_attention_q8_workspace_size(const FnQ8AttentionArgs *a, uint64_t *bytes, std::string &err) {
  if (bytes == nullptr) { err = "bytes is NULL"; return FNMOE_ERR_NULL; }
  if (const int rc = check(a, err)) return rc;
  *bytes = kWorkspaceBytes;
  return FNMOE_OK;
}

int paged_attention_q8(const FnQ8AttentionArgs *a, cudaStream_t s, std::string &err) {
  if (const int rc = check(a, err)) return rc;
  if (a->q_rows == 0) return FNMOE_OK;
  if (a->workspace == nullptr || a->workspace_bytes < kWorkspaceBytes) {
    err = "workspace needs " + std::to_string(kWorkspaceBytes) + " bytes";
    return FNMOE_ERR_WORKSPACE;
  }
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
  p.block = static_cast<int>(c.block);
  p.width = static_cast<int>(a->max_pages);
  p.pages = static_cast<int>(c.num_pages);
  p.scale = a->scale;
  const bool e4m3 = c.code_type == FNMOE_Q8_E4M3;
  switch (c.head_dim) {
    case 64: launch<64>(p, e4m3, s); break;
    case 128: launch<128>(p, e4m3, s); break;
    default: launch<256>(p, e4m3, s); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    err = std::string("paged attention q8: ") + cudaGetErrorString(e);
    return FNMOE_ERR_LAUNCH;
  }
  return FNMOE_OK;
}

}  // namespace fnmoe
