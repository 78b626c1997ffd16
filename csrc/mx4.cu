// Microscaled 4-bit floating point: rows are quantised, expanded and multiplied.
//
//   v[r, k] = e2m1(code[r, k]) * 2^(scale[r, k / 32] - 127)
//
// A code is a sign, two bits of exponent and one of mantissa (0, 1/2, 1, 3/2, 2, 3, 4, 6), two to a byte, the first in the low
// half; a scale is a power of two (e8m0) for 32 neighbours of a row, 255 for NaN. This is the format of the expert matrices of
// GPT-OSS checkpoints, which the reference hands to its GPU backends untouched (src/parallax/sglang/model_runner.py:358-366).
#include <cuda_fp4.h>

#include "common.cuh"
#include "mx4.cuh"
#include "pxl_api.h"

namespace {
using namespace pxl;

int check_launch() { return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA; }

// ---------------------------------------------------------------------------- rows -> codes and scales
// Four lanes per 32 values, eight values each. The scale is the smallest power of two that keeps the largest value within 6 (the
// largest e2m1 number), so that nothing is clipped; the values are then rounded to the nearest e2m1 number, ties to the even code.
// Powers of two make both steps exact but for that rounding. The largest value is found among the bit patterns, where NaN and
// infinities are the largest: a group that holds one becomes NaN (scale 255).
// Bound by memory: two groups per lane, both asked for first (25600 x 5120 in fp32 87 us, 6.8 TB/s, and 77 us in bf16; one each 95 and 81).
constexpr int kGroups = 2;
template <bool F32>
__global__ void __launch_bounds__(256) mx4_quant_rows_kernel(const void* __restrict__ x, int64_t ld, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales, int64_t total, int groups, int aligned) {
  pdl_wait();
  pdl_launch_dependents();
  const int l = threadIdx.x & 3;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (64 * kGroups) + (threadIdx.x >> 2);
  float v[kGroups][8];
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int64_t i = i0 + n * 64;
    const bool in = i < total;  // (whole fours of lanes; the others take part in the shuffles)
    int64_t at = in ? i * 32 : 0;
    if (ld != groups * 32 && in) {  // (a division of 64 bits takes as long as the rest)
      const int64_t row = i >> 32 ? i / groups : static_cast<uint32_t>(i) / static_cast<uint32_t>(groups);
      at = row * ld + (i - row * groups) * 32;
    }
    at += l * 8;
    if constexpr (F32) {
      const float* src = static_cast<const float*>(x) + at;
      if (aligned) {
        const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
        v[n][0] = a.x, v[n][1] = a.y, v[n][2] = a.z, v[n][3] = a.w, v[n][4] = b.x, v[n][5] = b.y, v[n][6] = b.z, v[n][7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] = src[j];
      }
    } else {
      const bf16* src = static_cast<const bf16*>(x) + at;
      if (aligned) {
        const bf16x8 w = ld_bf16x8(src);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_bf16x2(w.u[j]);
          v[n][2 * j] = f.x, v[n][2 * j + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] = __bfloat162float(src[j]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int64_t i = i0 + n * 64;
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[n][j]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // most = 1.f * 2^(p - 127) <= 6 * 2^e  <=>  e >= p - 129, or p - 128 for 1.f > 1.5
    const int p = static_cast<int>(most >> 23);
    const int e = max(-127, p - 129 + ((most & 0x7fffffu) > 0x400000u ? 1 : 0));
    const bool bad = p == 255;
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_fp4x2_storage_t b =
          __nv_cvt_float2_to_fp4x2(make_float2(v[n][2 * j] * inv, v[n][2 * j + 1] * inv), __NV_E2M1, cudaRoundNearest);
      packed |= static_cast<uint32_t>(b) << (8 * j);
    }
    if (i >= total) continue;
    reinterpret_cast<uint32_t*>(codes)[i * 4 + l] = bad ? 0u : packed;
    if (l == 0) scales[i] = static_cast<uint8_t>(bad ? 255 : e + 127);
  }
}

// ---------------------------------------------------------------------------- codes and scales -> values
__device__ __forceinline__ float mx4_power(uint32_t scale) {  // 2^(scale - 127)
  return scale == 255 ? __uint_as_float(0x7fc00000u) : scale == 0 ? __uint_as_float(0x400000u) : __uint_as_float(scale << 23);
}
__device__ __forceinline__ float2 mx4_pair(uint32_t byte) {  // the two numbers of a byte
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte & 255u), __NV_E2M1);
  return __half22float2(__half2(h));
}

constexpr int kWords = 4;
// Eight values per word, each exact in bf16 (down to its subnormals), but for those above its largest number. Bound by memory: four
// words per thread, all asked for first (25600 x 5120 53 us, 6.2 TB/s; one each 69).
__global__ void __launch_bounds__(256) mx4_expand_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              bf16* __restrict__ out, int64_t words) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (256 * kWords) + threadIdx.x;
  uint32_t w[kWords], s[kWords];
#pragma unroll
  for (int n = 0; n < kWords; ++n) {
    const int64_t i = i0 + n * 256;
    w[n] = i < words ? reinterpret_cast<const uint32_t*>(codes)[i] : 0;
    s[n] = i < words ? scales[i >> 2] : 0;
  }
#pragma unroll
  for (int n = 0; n < kWords; ++n) {
    const int64_t i = i0 + n * 256;
    if (i >= words) return;
    const float p = mx4_power(s[n]);
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = mx4_pair(w[n] >> (8 * j));
      o.u[j] = pack_bf16x2(f.x * p, f.y * p);
    }
    st_bf16x8(out + i * 8, o);
  }
}

// ---------------------------------------------------------------------------- weights laid out once (see mx4.cuh)
// A warp per row: the factor that its largest scale exceeds 128 by, NaN where it has a scale of 255.
__global__ void __launch_bounds__(256) mx4_row_scale_kernel(const uint8_t* __restrict__ scales, float* __restrict__ row_scale, int N,
                                                            int padded, int64_t rows, int groups) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int lane = threadIdx.x & 31, n = static_cast<int>(r % padded);
  int most = 0, nan = 0;
  if (n < N) {
    const uint8_t* s = scales + (r / padded * N + n) * groups;
    for (int g = lane; g < groups; g += 32) {
      const int v = s[g];
      if (v == 255) nan = 1;
      else most = max(most, v);
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) row_scale[r] = nan ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(127 + max(0, most - 128)) << 23);
}

__device__ __forceinline__ uint32_t mx4_place(uint32_t half) {  // four codes of a half word, where mx4_word takes them from
  const uint32_t a = half & 15u, b = half >> 4 & 15u, c = half >> 8 & 15u, d = half >> 12 & 15u;
  return (a >> 3) << 15 | (a & 7u) << 6 | (b >> 3) << 12 | (b & 7u) << 3 | (c >> 3) << 9 | (c & 7u) | (d >> 3) << 14 | (d & 6u) << 9 |
         (d & 1u) << 13;
}
// A thread per row of a block. (The powers of a row with a NaN scale are relative to the largest of its others too, which its factor
// does not say.) 51200 x 5120 95 us, the factors included: 2.9 TB/s, once per weight.
__global__ void __launch_bounds__(256) mx4_pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                       const float* __restrict__ row_scale, uint8_t* __restrict__ data, int N, int groups,
                                                       int n_blocks, int k_blocks) {
  pdl_wait();
  pdl_launch_dependents();
  const int r = threadIdx.x & 127, kb = blockIdx.x * 2 + (threadIdx.x >> 7), n_blk = blockIdx.y % n_blocks, n = n_blk * kTileRows + r;
  if (kb >= k_blocks) return;
  const int64_t expert = blockIdx.y / n_blocks, row = expert * N + n;
  uint8_t* const blk = data + ((expert * n_blocks + n_blk) * k_blocks + kb) * kBlockBytes;
  const float factor = row_scale[(expert * n_blocks + n_blk) * kTileRows + r];
  int over = static_cast<int>(__float_as_uint(factor) >> 23) - 127;
  if (isnan(factor)) {
    over = 0;
    for (int g = 0; g < groups; ++g) {
      const int v = scales[row * groups + g];
      if (v != 255) over = max(over, v - 128);
    }
  }
  uint32_t powers = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int g = kb * 4 + b;
    const bool in = n < N && g < groups;
    const int s = in ? scales[row * groups + g] : 0;
    const bool nan = s == 255;
    powers |= static_cast<uint32_t>(nan ? 255 : max(s - over, 0) + 126) << (8 * b);
    uint4 out = make_uint4(0, 0, 0, 0);
    if (in && (nan || s >= over)) {
      const uint4 c = *reinterpret_cast<const uint4*>(codes + (row * groups + g) * 16);
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // codes 0 .. 7 of a word: the even ones into the low half, the odd ones into the high half
        uint32_t even = 0, odd = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) even |= (w[j] >> (8 * i) & 15u) << (4 * i), odd |= (w[j] >> (8 * i + 4) & 15u) << (4 * i);
        o[j] = mx4_place(even) | mx4_place(odd) << 16;
      }
      out = make_uint4(o[0], o[1], o[2], o[3]);
    }
    *reinterpret_cast<uint4*>(blk + (b * kTileRows + r) * 16) = out;
  }
  *reinterpret_cast<uint32_t*>(blk + kCodeBytes + r * 4) = powers;
}

// ---------------------------------------------------------------------------- experts' rows
// out[t] = base[t] + sum_j w[t, j] y[pos_of[t, j]]: the experts' rows in fp32, so that a token's sum is rounded once. Bound by memory:
// 3001 tokens of eight rows of 2048 each 33 us, 6.3 TB/s.
__global__ void __launch_bounds__(256) moe_combine_f32_kernel(const float* __restrict__ y, const int* __restrict__ pos_of,
                                                              const float* __restrict__ w, const bf16* __restrict__ base,
                                                              bf16* __restrict__ out, int k, int H) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = blockIdx.x;
  for (int c = threadIdx.x * 4; c < H; c += 1024) {
    float a[4] = {};
    if (base) {
      const uint2 b = *reinterpret_cast<const uint2*>(base + t * H + c);
      const float2 f0 = unpack_bf16x2(b.x), f1 = unpack_bf16x2(b.y);
      a[0] = f0.x, a[1] = f0.y, a[2] = f1.x, a[3] = f1.y;
    }
    for (int j0 = 0; j0 < k; j0 += 4) {  // four rows in flight
      int p[4];
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = j0 + j < k ? pos_of[t * k + j0 + j] : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p[j] >= 0) v[j] = __ldcs(reinterpret_cast<const float4*>(y + static_cast<int64_t>(p[j]) * H + c));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (p[j] < 0) continue;
        const float f = w[t * k + j0 + j];
        a[0] += f * v[j].x, a[1] += f * v[j].y, a[2] += f * v[j].z, a[3] += f * v[j].w;
      }
    }
    *reinterpret_cast<uint2*>(out + t * H + c) = make_uint2(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]));
  }
}

}  // namespace

PXL_EXPORT int pxl_mx4_quant_rows(const void* x, int is_f32, int64_t ld, void* codes, void* scales, int64_t T, int K,
                                  cudaStream_t stream) {
  if (T < 0 || K <= 0 || K % 32) return PXL_ERR_INVALID_ARG;
  if (T == 0) return PXL_OK;
  const int groups = K / 32;
  const int64_t total = T * groups, blocks = ceil_div64(total, 64 * kGroups);
  if (blocks > 0x7fffffff) return PXL_ERR_TOO_LARGE;
  const int aligned = !(reinterpret_cast<uintptr_t>(x) & 15) && !(ld & (is_f32 ? 3 : 7));
  auto go = [&](auto kern) {
    pxl_host::launch(kern, static_cast<unsigned>(blocks), 256, 0, stream, x, ld, static_cast<uint8_t*>(codes),
                     static_cast<uint8_t*>(scales), total, groups, aligned);
  };
  if (is_f32) go(mx4_quant_rows_kernel<true>);
  else go(mx4_quant_rows_kernel<false>);
  return check_launch();
}

PXL_EXPORT int pxl_mx4_expand_rows(const void* codes, const void* scales, void* out, int64_t T, int K, cudaStream_t stream) {
  if (T < 0 || K <= 0 || K % 32) return PXL_ERR_INVALID_ARG;
  if (T == 0) return PXL_OK;
  const int64_t words = T * (K / 8), blocks = ceil_div64(words, 256 * kWords);
  if (blocks > 0x7fffffff) return PXL_ERR_TOO_LARGE;
  pxl_host::launch(mx4_expand_rows_kernel, static_cast<unsigned>(blocks), 256, 0, stream, static_cast<const uint8_t*>(codes),
                   static_cast<const uint8_t*>(scales), static_cast<bf16*>(out), words);
  pxl_host::next_launch_follows_whole();  // (the rows may be weights)
  return check_launch();
}

PXL_EXPORT int pxl_moe_combine_f32(const float* y, const int* pos_of, const float* w, const void* base, void* out, int T, int k,
                                   int H, cudaStream_t stream) {
  if (T < 0 || k <= 0 || H <= 0 || H % 8) return PXL_ERR_INVALID_ARG;
  // (rows are read and written in vectors of four)
  if ((reinterpret_cast<uintptr_t>(y) & 15) || ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(out)) & 7))
    return PXL_ERR_INVALID_ARG;
  if (T == 0) return PXL_OK;
  pxl_host::launch(moe_combine_f32_kernel, T, 256, 0, stream, y, pos_of, w, static_cast<const bf16*>(base), static_cast<bf16*>(out),
                   k, H);
  return check_launch();
}

PXL_EXPORT int pxl_mx4_pack(const void* codes, const void* scales, void* data, float* row_scale, int E, int N, int K, cudaStream_t stream) {
  if (E <= 0 || N <= 0 || K <= 0 || K % 32 || (reinterpret_cast<uintptr_t>(codes) & 15)) return PXL_ERR_INVALID_ARG;
  const int n_blocks = pxl::ceil_div(N, kTileRows), k_blocks = pxl::ceil_div(K, kTileCols), groups = K / 32;
  const int64_t rows = static_cast<int64_t>(E) * n_blocks * kTileRows;
  if (rows / 8 > 0x7fffffff) return PXL_ERR_TOO_LARGE;
  pxl_host::launch(mx4_row_scale_kernel, static_cast<unsigned>(rows / 8), 256, 0, stream, static_cast<const uint8_t*>(scales), row_scale, N,
                   n_blocks * kTileRows, rows, groups);
  // (the grid's second dimension ends at 65535: parts of whole experts' blocks of rows)
  const int per = 65535 / n_blocks;
  if (per < 1) return PXL_ERR_TOO_LARGE;
  for (int64_t e = 0; e < E; e += per) {
    const int n = static_cast<int>(E - e < per ? E - e : per);
    pxl_host::launch(mx4_pack_kernel, dim3(pxl::ceil_div(k_blocks, 2), n * n_blocks), 256, 0, stream,
                     static_cast<const uint8_t*>(codes) + e * N * groups * 16, static_cast<const uint8_t*>(scales) + e * N * groups,
                     row_scale + e * n_blocks * kTileRows, static_cast<uint8_t*>(data) + e * n_blocks * k_blocks * kBlockBytes, N, groups, n_blocks, k_blocks);
  }
  pxl_host::next_launch_follows_whole();
  return check_launch();
}
