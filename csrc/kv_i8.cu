// Keys and values in 8 bits: writing new tokens into such a cache, reading sequences out of it, thinning them out.
//
// A cache holds pages [blocks, Hkv, page, D] of int8 codes for K and as many for V, and kv_max fp32 [blocks, Hkv, 2]: the largest
// magnitude m of a page's keys and of its values. A code c stands for c * (m / 127). Codes are round(127 x / m), ties to even: 127 x is
// exact in fp32 for bf16 x and the quotient of two such numbers is no nearer than 2^-9 to a tie that it is not, so that the rounded
// quotient gives the code of the exact one. Tokens behind a page's first may raise m; the codes that are there become
// round(c * m_old / m_new), also from an exact product. m is NaN once a page was given a number that is not finite, until its first
// token is written again.
#include "common.cuh"
#include "pxl_api.h"

namespace {
using namespace pxl;

// round(127 x / m): both scaled down where 127 x would not fit; 0 for a page of zeros or without a magnitude
struct Coder {
  float m, up, safe;
  __device__ __forceinline__ explicit Coder(float m) : m(m) {
    up = m > 1.2676506e30f ? 127.f * 0x1p-64f : 127.f;
    safe = m > 1.2676506e30f ? m * 0x1p-64f : m > 0.f ? m : 1.f;
  }
  __device__ __forceinline__ int operator()(float x) const { return m == m ? __float2int_rn(__fdiv_rn(x * up, safe)) : 0; }
};
// round(c * from / to); as it is where the new magnitude is no number
struct Recoder {
  float from, to;
  __device__ __forceinline__ Recoder(float from, float to) : from(from), to(to) {
    if (to > 1.2676506e30f) this->from *= 0x1p-64f, this->to *= 0x1p-64f;
    if (to == 0.f) this->to = 1.f;
  }
  __device__ __forceinline__ int operator()(int c) const { return to == to ? __float2int_rn(__fdiv_rn(c * from, to)) : c; }
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (a & 0xff) | (b & 0xff) << 8 | (c & 0xff) << 16 | static_cast<uint32_t>(d) << 24;
}
__device__ __forceinline__ int code_of(uint32_t four, int i) { return static_cast<int8_t>(four >> (8 * i)); }

// ---- write ---------------------------------------------------------------------------------------------------------
// One CTA per (page that gets tokens, key head): warps 0 and 1 take the keys, 2 and 3 the values.
template <int D>
__global__ void __launch_bounds__(128)
store_kv_i8_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t k_stride, int64_t v_stride,
                   const int* __restrict__ block_tables, const int* __restrict__ cu_q, const int* __restrict__ ctx_lens,
                   int8_t* __restrict__ k_cache, int8_t* __restrict__ v_cache, float* __restrict__ kv_max, int T, int Hkv, int page,
                   int max_blocks, int64_t num_blocks, int* status) {
  constexpr int C = D / 8;  // chunks of 8 values in a row
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, kv = threadIdx.x >> 6, tid = threadIdx.x & 63;
  const int row0 = cu_q[b], n = cu_q[b + 1] - row0, t = ctx_lens[b];
  const int begin = t - n, from = begin > 0 ? begin : 0;
  const int p = from / page + static_cast<int>(blockIdx.x);
  if (n <= 0 || t <= 0 || p > (t - 1) / page) return;
  const int lo = from > p * page ? from - p * page : 0, hi = min(page, t - p * page);
  const int first = row0 + p * page + lo - begin;  // row of token lo of the page
  const int blk = p < max_blocks ? block_tables[static_cast<size_t>(b) * max_blocks + p] : -1;
  if (blk < 0 || blk >= num_blocks || first < 0 || first + hi - lo > T) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
    return;
  }
  const bf16* src = (kv ? v : k) + static_cast<int64_t>(first) * (kv ? v_stride : k_stride) + h * D;
  const int64_t stride = kv ? v_stride : k_stride;
  int8_t* dst = (kv ? v_cache : k_cache) + (static_cast<size_t>(blk) * Hkv + h) * page * D;
  float* m_at = kv_max + (static_cast<size_t>(blk) * Hkv + h) * 2 + kv;

  uint32_t top = 0;  // bits of the largest magnitude: ordered like the numbers, infinities and NaN above all of them
  for (int i = tid; i < (hi - lo) * C; i += 64) {
    const bf16x8 x = ld_bf16x8(src + (i / C) * stride + (i % C) * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, max(x.u[j] & 0x7fffu, (x.u[j] >> 16) & 0x7fffu));
  }
  __shared__ uint32_t tops[4];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  const float old = lo > 0 ? *m_at : 0.f;
  __syncthreads();
  top = max(tops[2 * kv], tops[2 * kv + 1]);
  const float now = top >= 0x7f80u || !(old == old) ? __uint_as_float(0x7fc00000u) : fmaxf(old, __uint_as_float(top << 16));
  if (tid == 0) *m_at = now;
  if (lo > 0 && now > old) {
    const Recoder again(old, now);
    for (int i = tid; i < lo * C; i += 64) {
      uint2 c = *reinterpret_cast<const uint2*>(dst + i * 8);
      uint32_t w[2] = {c.x, c.y};
#pragma unroll
      for (int j = 0; j < 2; ++j)
        w[j] = pack4(again(code_of(w[j], 0)), again(code_of(w[j], 1)), again(code_of(w[j], 2)), again(code_of(w[j], 3)));
      *reinterpret_cast<uint2*>(dst + i * 8) = make_uint2(w[0], w[1]);
    }
  }
  const Coder code(now);
  for (int i = tid; i < (hi - lo) * C; i += 64) {
    const bf16x8 x = ld_bf16x8(src + (i / C) * stride + (i % C) * 8);
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 a = unpack_bf16x2(x.u[2 * j]), c = unpack_bf16x2(x.u[2 * j + 1]);
      w[j] = pack4(code(a.x), code(a.y), code(c.x), code(c.y));
    }
    *reinterpret_cast<uint2*>(dst + lo * D + i * 8) = make_uint2(w[0], w[1]);
  }
}

// ---- read ----------------------------------------------------------------------------------------------------------
// A CTA takes 16 rows of the result, all heads, keys and values: 16 codes per thread and step.
constexpr int kLoadRows = 16;
template <int D>
__global__ void __launch_bounds__(256)
load_kv_i8_kernel(const int8_t* __restrict__ k_cache, const int8_t* __restrict__ v_cache, const float* __restrict__ kv_max,
                  const int* __restrict__ block_tables, const int* __restrict__ cu_k, bf16* __restrict__ k, bf16* __restrict__ v, int rows,
                  int B, int Hkv, int page, int max_blocks, int64_t num_blocks, int* status) {
  constexpr int C = D / 16;
  __shared__ int block_of[kLoadRows], place[kLoadRows];
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * kLoadRows;
  if (threadIdx.x < kLoadRows) {
    const int row = row0 + threadIdx.x;
    int blk = -1, off = 0;
    if (row < rows && row >= cu_k[0] && row < cu_k[B]) {
      int lo = 0, hi = B;  // the sequence: the last one that begins at or before the row
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu_k[mid] <= row) lo = mid;
        else hi = mid;
      }
      const int pos = row - cu_k[lo], p = pos / page;
      blk = p < max_blocks ? block_tables[static_cast<size_t>(lo) * max_blocks + p] : -1;
      off = pos % page;
      if (blk < 0 || blk >= num_blocks) {
        if (status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
        blk = -1;
      }
    }
    block_of[threadIdx.x] = blk;
    place[threadIdx.x] = off;
  }
  __syncthreads();
  const int per_row = 2 * Hkv * C, n = min(kLoadRows, rows - row0) * per_row;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = i / per_row, rest = i % per_row, kv = rest / (Hkv * C), h = rest / C % Hkv, c = rest % C;
    bf16* dst = (kv ? v : k) + (static_cast<size_t>(row0 + r) * Hkv + h) * D + c * 16;
    const int blk = block_of[r];
    uint4 x = make_uint4(0, 0, 0, 0);
    float scale = 0.f;
    if (blk >= 0) {
      const size_t head = static_cast<size_t>(blk) * Hkv + h;
      x = *reinterpret_cast<const uint4*>((kv ? v_cache : k_cache) + (head * page + place[r]) * D + c * 16);
      scale = __fdiv_rn(kv_max[head * 2 + kv], 127.f);
    }
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bf16x8 o[2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j >> 2].u[j & 3] = pack_bf16x2(code_of(w[j >> 1], 2 * (j & 1)) * scale, code_of(w[j >> 1], 2 * (j & 1) + 1) * scale);
    st_bf16x8(dst, o[0]);
    st_bf16x8(dst + 8, o[1]);
  }
}

// ---- thin out ------------------------------------------------------------------------------------------------------
// Which tokens stay. One CTA per (sequence, key head): the weight that the last of the chosen tokens has, by its bits from the top (11,
// 11 and 10 of them, a histogram each), then the tokens above it and the earliest of those that have it, in order: each warp counts and
// then writes those of its own stretch. The weights move to their new places chunk by chunk, the first chunk first: a token never
// moves back, so that no chunk writes where a later one reads.
constexpr int kPickThreads = 1024;
constexpr int kBins = 2048;

__device__ __forceinline__ uint32_t weight_key(float w) {  // ordered like the weights; NaN above all
  if (!(w == w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 is 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kPickThreads)
evict_pick_kernel(float* __restrict__ weights, int64_t W, int slots, const int* __restrict__ seq_slots, const int* __restrict__ ctx_lens,
                  int* __restrict__ kept, int* __restrict__ new_lens, int Hkv, int capacity, int keep, int recent, int first, int* status) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t sums[32], base_above[32], base_equal[32], found[2];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = seq_slots ? seq_slots[b] : b;
  int n = max(ctx_lens[b], 0);
  if (slot < 0 || slot >= slots || n > W || n > capacity) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, slot < 0 || slot >= slots ? PXL_DEV_BAD_SLOT : PXL_DEV_BAD_INDEX);
    n = 0;
  }
  float* w = weights + (static_cast<int64_t>(n > 0 ? slot : 0) * Hkv + h) * W;
  int* out = kept + (static_cast<int64_t>(b) * Hkv + h) * keep;
  const int stay = min(n, keep);
  if (h == 0 && threadIdx.x == 0) new_lens[b] = stay;
  if (n <= keep) {
    for (int i = threadIdx.x; i < keep; i += kPickThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int count = n - first - recent, want = keep - first - recent;  // of the tokens first .. first + count
  for (int i = threadIdx.x; i < first; i += kPickThreads) out[i] = i;
  for (int i = threadIdx.x; i < recent; i += kPickThreads) out[keep - recent + i] = n - recent + i;
  if (want > 0) {
    uint32_t prefix = 0, left = want;  // `left` of the keys that begin with `prefix` are chosen
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t above = pass == 0 ? 0 : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = threadIdx.x; i < kBins; i += kPickThreads) hist[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < count; i += kPickThreads) {
        const uint32_t key = weight_key(w[first + i]);
        if ((key & above) == prefix) atomicAdd(&hist[key >> shift & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // from the last bin down: two bins per thread, thread 0 the last two
      const uint32_t hi = hist[kBins - 1 - 2 * threadIdx.x], lo = hist[kBins - 2 - 2 * threadIdx.x];
      uint32_t incl = hi + lo;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
      if (warp == 0) {
        uint32_t s = sums[lane];
        const uint32_t own = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, s, d);
          if (lane >= d) s += up;
        }
        sums[lane] = s - own;
      }
      __syncthreads();
      const uint32_t before = sums[warp] + incl - hi - lo;
      if (before < left && left <= before + hi + lo) {
        const bool second = left > before + hi;
        found[0] = kBins - 1 - 2 * threadIdx.x - (second ? 1 : 0);
        found[1] = left - before - (second ? hi : 0);
      }
      __syncthreads();
      prefix |= found[0] << shift;
      left = found[1];
    }
    // `left` of the tokens whose key is `prefix`, all whose key is above it
    const int per = ceil_div(ceil_div(count, 32), 32) * 32, lo = min(warp * per, count), hi = min(lo + per, count);
    uint32_t above = 0, equal = 0;
    for (int i = lo + lane; i < hi; i += 32) {
      const uint32_t key = weight_key(w[first + i]);
      above += key > prefix;
      equal += key == prefix;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    __syncthreads();
    if (lane == 0) base_above[warp] = above, base_equal[warp] = equal;
    __syncthreads();
    uint32_t at = 0, ties = 0;  // chosen and equal ones before this warp's stretch
    for (int i = 0; i < warp; ++i) {
      const uint32_t e = base_equal[i];
      at += base_above[i] + (ties < left ? min(e, left - ties) : 0u);
      ties += e;
    }
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t key = i < hi ? weight_key(w[first + i]) : 0u;
      const uint32_t eq = __ballot_sync(0xffffffffu, i < hi && key == prefix), below = (1u << lane) - 1;
      const bool take = i < hi && (key > prefix || (key == prefix && ties + __popc(eq & below) < left));
      const uint32_t all = __ballot_sync(0xffffffffu, take);
      if (take) out[first + at + __popc(all & below)] = first + i;
      at += __popc(all);
      ties += __popc(eq);
    }
  }
  __syncthreads();
  for (int i0 = 0; i0 < keep; i0 += kPickThreads) {
    const int i = i0 + threadIdx.x;
    const float x = i < keep ? w[out[i]] : 0.f;
    __syncthreads();
    if (i < keep) w[i] = x;
    __syncthreads();
  }
  for (int i = keep + threadIdx.x; i < n; i += kPickThreads) w[i] = 0.f;
}

// The tokens that stay into their new pages: a CTA per (new page, key head), 16 codes per thread, PAGE * D / 16 threads for keys and
// as many for values at most; the new magnitude is the largest that a token of the page had.
template <int D, int PAGE>
__global__ void __launch_bounds__(256)
evict_move_kernel(int8_t* __restrict__ k_cache, int8_t* __restrict__ v_cache, float* __restrict__ kv_max, const int* __restrict__ block_tables,
                  const int* __restrict__ new_tables, const int* __restrict__ kept, const int* __restrict__ new_lens, int Hkv, int max_blocks,
                  int max_new, int64_t num_blocks, int keep, int* status) {
  constexpr int C = D / 16, kSteps = 2 * PAGE * C / 256 > 0 ? 2 * PAGE * C / 256 : 1;
  __shared__ int block_of[PAGE], place[PAGE];
  __shared__ float most[2][PAGE];
  pdl_wait();
  pdl_launch_dependents();
  const int p = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int n = min(PAGE, new_lens[b] - p * PAGE);
  if (n <= 0) return;
  const int to = p < max_new ? new_tables[static_cast<size_t>(b) * max_new + p] : -1;
  if (to < 0 || to >= num_blocks) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
    return;
  }
  if (threadIdx.x < PAGE) {
    float mk = 0.f, mv = 0.f;
    int blk = -1, off = 0;
    if (threadIdx.x < n) {
      const int i = kept[(static_cast<int64_t>(b) * Hkv + h) * keep + p * PAGE + threadIdx.x];
      blk = i / PAGE < max_blocks ? block_tables[static_cast<size_t>(b) * max_blocks + i / PAGE] : -1;
      off = i % PAGE;
      if (blk < 0 || blk >= num_blocks) {
        if (status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
        blk = -1;
      } else {
        const float2 m = *reinterpret_cast<const float2*>(kv_max + (static_cast<size_t>(blk) * Hkv + h) * 2);
        mk = m.x, mv = m.y;
      }
    }
    block_of[threadIdx.x] = blk;
    place[threadIdx.x] = off;
    most[0][threadIdx.x] = mk;
    most[1][threadIdx.x] = mv;
  }
  __syncthreads();
  float top[2] = {0.f, 0.f};
  for (int i = 0; i < PAGE; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j) top[j] = top[j] == top[j] && !(most[j][i] <= top[j]) ? most[j][i] : top[j];  // (NaN stays)
  }
  const size_t dst = (static_cast<size_t>(to) * Hkv + h) * PAGE;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = s * 256 + threadIdx.x, kv = i / (PAGE * C), r = i / C % PAGE, c = i % C;
    if (kv > 1 || r >= n || block_of[r] < 0) continue;
    int8_t* cache = kv ? v_cache : k_cache;
    const uint4 x = *reinterpret_cast<const uint4*>(cache + ((static_cast<size_t>(block_of[r]) * Hkv + h) * PAGE + place[r]) * D + c * 16);
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    const float m = most[kv][r], t = top[kv];
    if (m != t) {
      const Recoder again(m, t);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = pack4(again(code_of(w[j], 0)), again(code_of(w[j], 1)), again(code_of(w[j], 2)), again(code_of(w[j], 3)));
    }
    *reinterpret_cast<uint4*>(cache + (dst + r) * D + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (threadIdx.x < 2) kv_max[(static_cast<size_t>(to) * Hkv + h) * 2 + threadIdx.x] = threadIdx.x ? top[1] : top[0];
}

bool cache_ok(int Hkv, int D, int page, int max_blocks, int64_t num_blocks, const void* k_cache, const void* v_cache) {
  return Hkv > 0 && (D == 64 || D == 128) && (page == 16 || page == 32 || page == 64) && max_blocks > 0 && num_blocks > 0 &&
         num_blocks * Hkv * page < (1ll << 31) && !((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15);
}
int done() { return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA; }

}  // namespace

PXL_EXPORT int pxl_kv_i8_store(const void* k, const void* v, int64_t k_stride, int64_t v_stride, const int* block_tables, const int* cu_q,
                               const int* ctx_lens, void* k_cache, void* v_cache, float* kv_max, int T, int B, int max_q_len, int Hkv, int D,
                               int page, int max_blocks, int64_t num_blocks, int* status, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || max_q_len <= 0) return PXL_OK;
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || Hkv > 65535 || (k_stride & 7) || (v_stride & 7) ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
    return PXL_ERR_INVALID_ARG;
  if (B > 65535) return PXL_ERR_TOO_LARGE;
  const dim3 grid((max_q_len + page - 2) / page + 1, Hkv, B);
  auto go = [&](auto kernel) {
    pxl_host::launch(kernel, grid, dim3(128), 0, stream, static_cast<const bf16*>(k), static_cast<const bf16*>(v), k_stride, v_stride,
                     block_tables, cu_q, ctx_lens, static_cast<int8_t*>(k_cache), static_cast<int8_t*>(v_cache), kv_max, T, Hkv, page,
                     max_blocks, num_blocks, status);
    return done();
  };
  return D == 64 ? go(store_kv_i8_kernel<64>) : go(store_kv_i8_kernel<128>);
}

PXL_EXPORT int pxl_kv_i8_load(const void* k_cache, const void* v_cache, const float* kv_max, const int* block_tables, const int* cu_k, void* k,
                              void* v, int rows, int B, int Hkv, int D, int page, int max_blocks, int64_t num_blocks, int* status,
                              cudaStream_t stream) {
  if (rows <= 0) return PXL_OK;
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || B < 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
    return PXL_ERR_INVALID_ARG;
  auto go = [&](auto kernel) {
    pxl_host::launch(kernel, dim3(ceil_div(rows, kLoadRows)), dim3(256), 0, stream, static_cast<const int8_t*>(k_cache),
                     static_cast<const int8_t*>(v_cache), kv_max, block_tables, cu_k, static_cast<bf16*>(k), static_cast<bf16*>(v), rows, B,
                     Hkv, page, max_blocks, num_blocks, status);
    return done();
  };
  return D == 64 ? go(load_kv_i8_kernel<64>) : go(load_kv_i8_kernel<128>);
}

PXL_EXPORT int pxl_kv_i8_evict(void* k_cache, void* v_cache, float* kv_max, float* weights, int64_t W, int slots, const int* seq_slots,
                               const int* block_tables, const int* ctx_lens, const int* new_tables, int* kept, int* new_lens, int B, int Hkv,
                               int D, int page, int max_blocks, int max_new, int64_t num_blocks, int keep, int recent, int first, int* status,
                               cudaStream_t stream) {
  if (B <= 0) return PXL_OK;
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || max_new <= 0 || W <= 0 || keep < 1 || recent < 0 || first < 0 ||
      static_cast<int64_t>(recent) + first > keep || keep > static_cast<int64_t>(max_new) * page || static_cast<int64_t>(max_blocks) * page > INT32_MAX)
    return PXL_ERR_INVALID_ARG;
  if (B > 65535 || Hkv > 65535) return PXL_ERR_TOO_LARGE;
  pxl_host::launch(evict_pick_kernel, dim3(Hkv, B), dim3(kPickThreads), 0, stream, weights, W, slots, seq_slots, ctx_lens, kept, new_lens, Hkv,
                   max_blocks * page, keep, recent, first, status);
  if (const int rc = done()) return rc;
  auto go = [&](auto kernel) {
    pxl_host::launch(kernel, dim3(ceil_div(keep, page), Hkv, B), dim3(256), 0, stream, static_cast<int8_t*>(k_cache),
                     static_cast<int8_t*>(v_cache), kv_max, block_tables, new_tables, kept, new_lens, Hkv, max_blocks, max_new, num_blocks,
                     keep, status);
    pxl_host::next_launch_follows_whole();  // the new lengths
    return done();
  };
  if (D == 64) return page == 16 ? go(evict_move_kernel<64, 16>) : page == 32 ? go(evict_move_kernel<64, 32>) : go(evict_move_kernel<64, 64>);
  return page == 16 ? go(evict_move_kernel<128, 16>) : page == 32 ? go(evict_move_kernel<128, 32>) : go(evict_move_kernel<128, 64>);
}
