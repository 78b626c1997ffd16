// Codes of an 8-bit cache (kv_i8.cu) as f16 numbers, and what the attention kernels over it share.
#pragma once

#include "common.cuh"

namespace pxl {

// Bytes of four codes with their sign bits flipped (u = code + 128), two of them put under the exponent of 1024: 1024 + u, exactly; minus
// 1152 that is the code. One operation for two numbers and half a flip: int8 has no conversion of its own to 16-bit floats.
__device__ __forceinline__ uint32_t flip_codes(uint32_t four) { return four ^ 0x80808080u; }
template <uint32_t SELECT>  // bytes of the flipped word in the low halves of the two numbers: 0x4x4y
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t flipped) {
  const uint32_t raw = __byte_perm(flipped, 0x64646464u, SELECT);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(raw), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ void mma_m16n8k16_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Power of two that brings a row's largest magnitude into [2^13, 2^14), and its inverse: bf16 numbers down to 2^-27 of it stay exact in
// f16 (below, they lose bits that the fp32 sums of the products would lose as well).
__device__ __forceinline__ float row_up(float most, float& down) {
  int up = 267 - static_cast<int>(__float_as_uint(most) >> 23);
  up = up < 1 ? 1 : up > 253 ? 253 : up;
  down = __uint_as_float(static_cast<uint32_t>(254 - up) << 23);
  return __uint_as_float(static_cast<uint32_t>(up) << 23);
}
constexpr float kInv127 = 1.f / 127.f;

// share of a magnitude in the largest so far; 0 of none
__device__ __forceinline__ float page_share(float m, float most) {
  if (most > 1e-30f && most < 1e30f) return __fdividef(m, most);  // (which is 0 for a divisor above 2^126)
  return m == 0.f ? 0.f : __fdiv_rn(m, most);
}

// log2 of that, from log2 of the largest; not below -40 (whose values are lost beside the others'); 0 without a magnitude, so that the sums
// of exponentials, and the weights with them, depend on the keys alone
__device__ __forceinline__ float page_log(float m, float log_most) { return m == m ? fmaxf(__log2f(m) - log_most, -40.f) : 0.f; }

}  // namespace pxl

namespace pxl_host {

// The second kernel of an operator: its launch carries the attribute whether the caller is in a chain or not. The kernel before it is the
// operator's own and waited for what ran ahead of it before it let this one begin.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_behind(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  int& state = launch_chain();
  const int was = state;
  state = kInChain;
  const cudaError_t rc = launch(kern, grid, block, smem, stream, static_cast<Args&&>(args)...);
  state = was;
  return rc;
}

// Tensor map of the codes [rows, D] int8 with boxes of one page, swizzled by their row's width.
inline bool make_tmap_codes(CUtensorMap* out, const void* base, uint64_t rows, int D, int page) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), rows};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(D)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(D), static_cast<cuuint32_t>(page)};
  cuuint32_t estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries [T, Hq, D] as boxes of tokens x heads of a key head x 64 columns.
inline bool make_tmap_queries(CUtensorMap* out, const void* q, int64_t q_stride, int T, int Hq, int D, int G) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(T)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(T > 1 ? q_stride : static_cast<int64_t>(Hq) * D) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(128 / G)};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace pxl_host
