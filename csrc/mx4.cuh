// What the kernels of microscaled 4-bit numbers share.
#pragma once

#include "common.cuh"
#include "pxl_api.h"

namespace pxl {

// Weights of pxl_gemm_mx4 are laid out once, in blocks of 128 rows x 128 columns that lie one behind the other along a row of
// blocks: 8192 bytes of codes [column group of 32][row][16 bytes], then 512 bytes of powers [row][column group]. Rows and columns
// are filled up to a whole block with zeros. Within a word of eight codes the bits are placed so that two numbers at a time become
// bf16 with few instructions: the even numbers' bits are in the low half of the word, the odd ones' in the high half, and
//
//   number of the half   0           1           2          3
//   sign at bit          15          12          9          14
//   magnitude at bits    8 .. 6      5 .. 3      2 .. 0     11, 10 and 13
//
// A sign at bit 15 and a magnitude at 8 .. 6 is the bf16 of the number times 2^-126 (1/2 is a subnormal there), and one product
// with a power of two makes it the value: exact. The stored power is the exponent field of 2^(scale - 1), for scales up to 128; the
// rows' factors hold what a row with a larger scale exceeds that by, and NaN for a row with a scale of 255.
constexpr int kTileRows = 128, kTileCols = 128;
constexpr int kCodeBytes = kTileRows * kTileCols / 2, kBlockBytes = kCodeBytes + kTileRows * 4;

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Factors of the shifts to the left, as arguments of the kernel: multiplications of unknown factors run on the FMA pipe, where the
// compiler would put shifts on the ALU, whose rate bounds the expansion.
struct Mx4Shift {
  uint32_t by1, by3, by6;  // 2, 8, 64
};
constexpr Mx4Shift kMx4Shift{2u, 8u, 64u};
// eight codes as placed above, and the power's exponent field in both halves -> eight values in bf16
__device__ __forceinline__ void mx4_word(uint32_t w, uint32_t power2, const Mx4Shift& s, uint32_t (&o)[4]) {
  o[0] = mul_bf16x2(w & 0x81c081c0u, power2);
  o[1] = mul_bf16x2((w * s.by3) & 0x81c081c0u, power2);
  o[2] = mul_bf16x2((w * s.by6) & 0x81c081c0u, power2);
  o[3] = mul_bf16x2(((w * s.by1) & 0x80008000u) | ((w >> 3) & 0x01800180u) | ((w >> 7) & 0x00400040u), power2);
}
// byte h of four powers in the exponent fields of both halves
__device__ __forceinline__ uint32_t mx4_power2(uint32_t four, int h) { return __byte_perm(four, 0, 0x4040 | h | h << 8) << 7; }

__device__ __forceinline__ float mx4_gate(float g, float u, int epi, float limit) {
  float s = g;
  if (epi == PXL_EPI_CLIP_GLU) {
    g = g > limit ? limit : g;
    u = u < -limit ? -limit : u > limit ? limit : u;
    s = 1.702f * g;
    u += 1.f;
  }
  return __fdividef(g, 1.f + __expf(-s)) * u;
}

}  // namespace pxl

namespace pxl_host {
// gemv_mx4.cu: what pxl_gemm_mx4 does, for up to four rows; whether that is the faster way for them
bool gemv_mx4_takes(int M, int N, int K);
int gemv_mx4(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc, const void* bias,
             const void* residual, int64_t ldr, int M, int N, int K, int epi, float limit, cudaStream_t stream);
}  // namespace pxl_host
