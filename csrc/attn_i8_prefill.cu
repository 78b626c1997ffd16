// Attention over keys and values in 8 bits (layout: kv_i8.cu): one CTA per (query row, key head), a thread per key for the scores and per
// column for the output.
#include "common.cuh"
#include "pxl_api.h"

namespace {
using namespace pxl;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxGroup = 16, kKeys = 128;

struct Cache {
  const int8_t *k, *v;
  const float* kv_max;
  const int* block_tables;
  int Hkv, page, max_blocks;
  int64_t num_blocks;
  int* status;

  // row of token t of sequence b (whose codes and magnitude are found by it); -1 off the cache
  __device__ __forceinline__ int64_t row(int b, int t, int h) const {
    const int p = t / page, blk = p < max_blocks ? block_tables[static_cast<size_t>(b) * max_blocks + p] : -1;
    if (blk < 0 || blk >= num_blocks) {
      if (status) atomicCAS(status, 0, PXL_DEV_BAD_BLOCK_DECODE);
      return -1;
    }
    return (static_cast<int64_t>(blk) * Hkv + h) * page + t % page;
  }
};

template <int D>
__device__ __forceinline__ float dot(const int8_t* k, const float* q) {
  float s = 0.f;
  for (int c = 0; c < D; c += 16) {
    const int4 x = *reinterpret_cast<const int4*>(k + c);
    const int w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) s = fmaf(static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3))), q[c + j], s);
  }
  return s;
}

template <int D>
__global__ void __launch_bounds__(128)
attn_i8_kernel(const bf16* __restrict__ q, int64_t q_stride, const Cache cache, const int* __restrict__ cu_q, const int* __restrict__ ctx_lens,
               bf16* __restrict__ out, int64_t out_stride, const float* __restrict__ sinks, float* __restrict__ lse, int B, int Hq,
               float scale_log2, int window) {
  __shared__ float q_sm[kMaxGroup][D], p_sm[kMaxGroup][kKeys], m_sm[4], l_sm[4];
  __shared__ int64_t row_sm[kKeys];
  __shared__ float M[kMaxGroup], L[kMaxGroup];
  const int row = blockIdx.x, h = blockIdx.y, G = Hq / cache.Hkv, tid = threadIdx.x, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  int b = row, pos = ctx_lens[cu_q ? 0 : row] - 1;
  if (cu_q) {
    if (row < cu_q[0] || row >= cu_q[B]) return;
    b = 0;
    while (cu_q[b + 1] <= row) ++b;
    pos = ctx_lens[b] - cu_q[b + 1] + row;
  }
  const int hi = pos + 1, lo = window > 0 && hi > window ? hi - window : 0;
  for (int i = tid; i < G * D; i += 128)
    q_sm[i / D][i % D] = __bfloat162float(q[row * q_stride + (h * G + i / D) * D + i % D]) * scale_log2;
  __syncthreads();
  auto score = [&](int64_t at, int g) {
    return dot<D>(cache.k + at * D, q_sm[g]) * (cache.kv_max[at / cache.page * 2] * (1.f / 127.f));
  };
  for (int g = 0; g < G; ++g) {
    float m = -INFINITY, l = 0.f;
    for (int t = lo + tid; t < hi; t += kKeys) {
      const int64_t at = cache.row(b, t, h);
      if (at < 0) continue;
      const float s = score(at, g), mn = fmaxf(m, s);
      l = l * exp2f(m - mn) + exp2f(s - mn);
      m = mn;
    }
    const float wm = warp_reduce_max(m);
    l = warp_reduce_sum(m == -INFINITY ? 0.f : l * exp2f(m - wm));
    if ((tid & 31) == 0) m_sm[warp] = wm, l_sm[warp] = l;
    __syncthreads();
    if (tid == 0) {
      float top = sinks ? sinks[h * G + g] * kLog2e : -INFINITY;
      const float sink = top;
      for (int i = 0; i < 4; ++i) top = fmaxf(top, m_sm[i]);
      float sum = sinks ? exp2f(sink - top) : 0.f;
      for (int i = 0; i < 4; ++i) sum += m_sm[i] == -INFINITY ? 0.f : l_sm[i] * exp2f(m_sm[i] - top);
      M[g] = top;
      L[g] = sum;
      if (lse) lse[static_cast<size_t>(row) * Hq + h * G + g] = sum > 0.f || !(sum == sum) ? top + log2f(sum) : INFINITY;
    }
    __syncthreads();
  }
  float acc[kMaxGroup];
  for (int g = 0; g < G; ++g) acc[g] = 0.f;
  for (int t0 = lo; t0 < hi; t0 += kKeys) {
    const int64_t at = t0 + tid < hi ? cache.row(b, t0 + tid, h) : -1;
    __syncthreads();
    row_sm[tid] = at;
    const float vs = at < 0 ? 0.f : cache.kv_max[at / cache.page * 2 + 1] * (1.f / 127.f);
    for (int g = 0; g < G; ++g) p_sm[g][tid] = at < 0 ? 0.f : exp2f(score(at, g) - M[g]) * vs;
    __syncthreads();
    if (tid < D) {
      for (int j = 0; j < kKeys; ++j) {
        if (row_sm[j] < 0) continue;
        const float x = cache.v[row_sm[j] * D + tid];
        for (int g = 0; g < G; ++g) acc[g] = fmaf(p_sm[g][j], x, acc[g]);
      }
    }
  }
  if (tid < D)
    for (int g = 0; g < G; ++g)
      out[row * out_stride + (h * G + g) * D + tid] = __float2bfloat16(L[g] > 0.f || !(L[g] == L[g]) ? acc[g] / L[g] : 0.f);
}

// What each token got: a thread per key goes through the queries that see it.
template <int D>
__global__ void __launch_bounds__(128)
attn_i8_weights_kernel(const bf16* __restrict__ q, int64_t q_stride, const Cache cache, const int* __restrict__ cu_q,
                       const int* __restrict__ ctx_lens, const float* __restrict__ lse, float* __restrict__ weights, int64_t W, int slots,
                       const int* __restrict__ seq_slots, int Hq, float scale_log2, int window) {
  __shared__ float q_sm[kMaxGroup][D];
  const int b = blockIdx.z, h = blockIdx.y, G = Hq / cache.Hkv, t = blockIdx.x * kKeys + threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = cu_q ? cu_q[b] : b, n = cu_q ? cu_q[b + 1] - row0 : 1, ctx = ctx_lens[b];
  const int slot = seq_slots ? seq_slots[b] : b;
  if (n <= 0 || static_cast<int>(blockIdx.x) * kKeys >= ctx) return;
  if (slot < 0 || slot >= slots || ctx > W) {
    if (threadIdx.x == 0 && cache.status) atomicCAS(cache.status, 0, slot < 0 || slot >= slots ? PXL_DEV_BAD_SLOT : PXL_DEV_BAD_INDEX);
    return;
  }
  const int64_t at = t < ctx ? cache.row(b, t, h) : -1;
  const float ks = at < 0 ? 0.f : cache.kv_max[at / cache.page * 2] * (1.f / 127.f);
  float sum = 0.f;
  for (int r = 0; r < n; ++r) {
    const int pos = ctx - n + r;
    if (pos < static_cast<int>(blockIdx.x) * kKeys) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < G * D; i += 128)
      q_sm[i / D][i % D] = __bfloat162float(q[(row0 + r) * q_stride + (h * G + i / D) * D + i % D]) * scale_log2;
    __syncthreads();
    if (at >= 0 && t <= pos && (window <= 0 || t > pos - window))
      for (int g = 0; g < G; ++g) sum += exp2f(dot<D>(cache.k + at * D, q_sm[g]) * ks - lse[static_cast<size_t>(row0 + r) * Hq + h * G + g]);
  }
  if (at >= 0) weights[(static_cast<int64_t>(slot) * cache.Hkv + h) * W + t] += sum;
}

}  // namespace

PXL_EXPORT int64_t pxl_attn_i8_prefill_workspace(int T, int B, int max_q_len, int Hq, int Hkv, int D, int max_ctx, int with_weights) {
  return with_weights ? static_cast<int64_t>(T) * Hq * 4 : 0;
}

PXL_EXPORT int pxl_attn_i8_prefill(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const float* kv_max,
                           const int* block_tables, const int* cu_q, const int* ctx_lens, void* out, int64_t out_stride, const float* sinks,
                           float* weights, int64_t W, int slots, const int* seq_slots, void* workspace, int64_t workspace_bytes, int T, int B,
                           int max_q_len, int Hq, int Hkv, int D, int page, int max_blocks, int64_t num_blocks, float scale, int window,
                           int max_ctx, int* status, cudaStream_t stream) {
  if (T <= 0 || B <= 0) return PXL_OK;
  if ((D != 64 && D != 128) || (page != 16 && page != 32 && page != 64) || Hkv <= 0 || Hq % Hkv || Hq / Hkv > kMaxGroup || !(scale > 0.f) ||
      (q_stride & 7) || (out_stride & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) || max_blocks <= 0 || num_blocks <= 0 ||
      num_blocks * Hkv * page >= (1ll << 31) || workspace_bytes < pxl_attn_i8_prefill_workspace(T, B, max_q_len, Hq, Hkv, D, max_ctx, weights != nullptr))
    return PXL_ERR_INVALID_ARG;
  if (Hkv > 65535 || B > 65535) return PXL_ERR_TOO_LARGE;
  const Cache cache{static_cast<const int8_t*>(k_cache), static_cast<const int8_t*>(v_cache), kv_max, block_tables, Hkv, page, max_blocks,
                    num_blocks, status};
  float* lse = weights ? static_cast<float*>(workspace) : nullptr;
  auto go = [&](auto attend, auto weigh) {
    pxl_host::launch(attend, dim3(T, Hkv), dim3(128), 0, stream, static_cast<const bf16*>(q), q_stride, cache, cu_q, ctx_lens,
                     static_cast<bf16*>(out), out_stride, sinks, lse, B, Hq, scale * kLog2e, window);
    if (weights)
      pxl_host::launch(weigh, dim3(ceil_div(max_ctx, kKeys), Hkv, B), dim3(128), 0, stream, static_cast<const bf16*>(q), q_stride, cache, cu_q,
                       ctx_lens, lse, weights, W, slots, seq_slots, Hq, scale * kLog2e, window);
    return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
  };
  return D == 64 ? go(attn_i8_kernel<64>, attn_i8_weights_kernel<64>) : go(attn_i8_kernel<128>, attn_i8_weights_kernel<128>);
}
