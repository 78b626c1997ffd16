// Attention of new tokens over keys and values in 8 bits (layout: kv_i8.cu) on the 5th-generation tensor cores.
//
// A CTA takes 128 / G tokens of a sequence twice (G query heads of a key head: G rows per token, two units of 128 rows) and a range of
// its keys in tiles of 128:
//   warp 8      : TMA producer. The queries once (a box of tokens x heads x 64 columns per unit and half), then the codes of K and V of a
//                 tile, page by page, into a ring of staging tiles; and what the softmax needs to know of the tile's pages.
//   warps 12-15 : convert the codes to f16 tiles, K-major for K, MN-major for V, in a ring that the tensor cores read: once for the 256
//                 rows of both units.
//   warp 9      : MMA issuer. P_u V, then S_u = Q_u K^T of the next tile, u = 0, 1 in turn: the products of one unit run under the softmax
//                 of the other.
//   warps 0-7   : softmax, a row of 128 scores per thread. First they scale their rows of Q by powers of two into f16. P replaces S in
//                 tensor memory as f16, the A operand of the second product.
// A score is multiplied by its page's key magnitude with the softmax scale. Values are held relative to R, at least the largest value
// magnitude so far and at most twice as much when it was chosen: an exponential is taken of the score plus log2 of the page's share of R, so
// that what is rounded to f16 is the probability times the share (2^-11 of it, down to 2^-21 of the row's largest; 2^-32 below), and the
// sum of a page's 16 columns is divided by the share again. Both the reference maximum (by 2^8) and R are let run ahead before O in tensor
// memory is rescaled. R is one for the CTA, unless that is more than 16 times what a row has seen of its own (a page that only others see is far
// above the rest): then the row keeps one for itself.
// 8111 tokens, 32 heads, D = 128, twice: 757 us, 0.92 PFLOP/s (739 to 787 by run and card). A tile takes 4400 clocks for both units, the chain of one unit's: product 550,
// softmax 2700, notice and issue 1000; the tensor pipe is 41 % full. Two units of 128 rows for one conversion: with one the converting warps
// would take as long as the softmax. (Heads of 64: CTAs of one unit, two on an SM, take longer too, 288 us for 239 of 5 x 3001 tokens with
// windows of 128, 802 for 674 of the two prompts. Since rows have an R of their own where that is needed, 238 and 677.)
// Few rows: the keys are split over several CTAs, whose results a second kernel adds up.
// Every wait is bounded; on expiry the kernel records a status code, all roles unwind, tensor memory is freed.
#include <atomic>

#include "attention_rows.cuh"
#include "attention_walk.cuh"
#include "common.cuh"
#include "kv_i8.cuh"
#include "pxl_api.h"
#include "tc_issue.cuh"

namespace {
using namespace pxl;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kT = 128;  // keys per tile
constexpr int kRowsQ = 128;
constexpr int kProducerWarp = 8, kMmaWarp = 9, kConvertWarp = 12, kThreads = 512;
constexpr int kHalf = 128 * 128;  // bytes of 64 columns of 128 rows
constexpr float kUp = 7.f;        // log2 of the factor on probabilities; 2^8 of a stale maximum on top stays below 2^16
constexpr int kRing = 8;          // tiles whose pages' numbers are kept: the producer is at most three ahead of a softmax, five at D = 64

template <int D>
struct Shape {
  static constexpr int kTile = D / 64 * kHalf;         // a f16 tile of 128 rows
  static constexpr int kCodes = 128 * D;               // codes of a tile
  static constexpr int kStages = D == 128 ? 2 : 4;     // staging tiles
  static constexpr int kSlots = D == 128 ? 4 : 6;      // f16 tiles
  static constexpr int kOffKV = 2 * kTile;             // behind the two units of Q
  static constexpr int kOffCodes = kOffKV + kSlots * kTile;
  static constexpr int kOffPages = kOffCodes + kStages * kCodes;  // [kRing][8] float4
  static constexpr int kOffMags = kOffPages + kRing * 8 * 16;     // [kRing][8] magnitudes of values
  static constexpr int kOffBars = kOffMags + kRing * 8 * 4;
  static constexpr int kSmem = 1024 + kOffBars + 256;
  static constexpr uint32_t kIdescS = umma_idesc(kRowsQ, kT, 0, 0);
  static constexpr uint32_t kIdescPV = umma_idesc(kRowsQ, D, 0, 0) | (1u << 16);  // B (V) is MN-major
};
static_assert(Shape<128>::kSmem <= 232448);

struct Args {
  const float2* kv_max;
  const int *block_tables, *cu_q, *ctx_lens;
  bf16* out;
  int64_t out_stride;
  const float* sinks;
  float *lse, *parts;  // log2 of the sums [T, Hq] (null: not wanted); partial results [splits][T * Hq][D + 4]
  int T, max_q_len, Hq, Hkv, page, max_blocks;
  int64_t num_blocks;
  float scale_log2;
  int window, splits;
  int* status;
};

// What a row's keys gave: output in units of R times 2^kUp, maximum (log2), sum, R, whether it saw values without a magnitude.
constexpr int kPartTail = 4;

// V tile as B operand of all its columns: 64-column chunks kHalf apart
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  return (umma_desc_k_sw128(addr) & ~(0x3fffull << 16)) | (static_cast<uint64_t>(kHalf >> 4) << 16);
}

// One tile of 128 codes x D into f16. Eight neighbouring lanes take four chunks of 16 codes of rows r and r ^ 5: both the chunk that is
// read and the two that are written fall on all banks.
template <int D>
__device__ __forceinline__ void convert_tile(uint32_t codes, uint32_t tile, int warp, int lane) {
  constexpr int kSteps = D / 16;  // 8 rows x 4 chunks at a time, 16 * D / 64 of them for four warps
  const int c4 = lane & 3, r8 = (lane >> 3) ^ ((lane & 4) ? 5 : 0);
#pragma unroll
  for (int s0 = 0; s0 < kSteps; s0 += 4) {
    uint32_t w[4][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int i = (s0 + s) * 4 + warp, half = D == 128 ? i & 1 : 0, row = (D == 128 ? i >> 1 : i) * 8 + r8, c = half * 4 + c4;
      const uint32_t at = D == 128 ? row * 128 + ((c ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[s][0]), "=r"(w[s][1]), "=r"(w[s][2]), "=r"(w[s][3])
                   : "r"(codes + at));
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int i = (s0 + s) * 4 + warp, half = D == 128 ? i & 1 : 0, row = (D == 128 ? i >> 1 : i) * 8 + r8;
      const uint32_t at = tile + half * kHalf + row * 128;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t a = flip_codes(w[s][2 * p]), b = flip_codes(w[s][2 * p + 1]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((c4 * 2 + p) ^ (row & 7)) << 4)), "r"(codes_f16x2<0x4140>(a)),
                     "r"(codes_f16x2<0x4342>(a)), "r"(codes_f16x2<0x4140>(b)), "r"(codes_f16x2<0x4342>(b))
                     : "memory");
      }
    }
  }
}

// This thread's row of Q in f16, in place, scaled by a power of two; returns the inverse of that. 0 for a row that is nobody's.
template <int D>
__device__ __forceinline__ float convert_row(uint32_t row_addr, int r, bool valid) {
  float most = 0.f;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    uint32_t x[4];
    const uint32_t at = row_addr + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(x[j]);
      most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
  }
  float down;
  const float up = row_up(most, down);
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    uint32_t x[4];
    const uint32_t at = row_addr + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(x[j]);
      x[j] = valid ? pack_f16x2(f.x * up, f.y * up) : 0u;
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
  }
  return down;
}

// Which columns of a tile the rows of a warp see: [from, to) of this lane's row; of the 16-column groups, those that some row sees some of
// and those that all rows see whole, a bit each.
struct Seen {
  int from = 0, to = kT;
  uint32_t some = 0xffu, whole = 0xffu;
  Seen() = default;
  __device__ __forceinline__ Seen(int from, int to) : from(from), to(to) {
    const int f_min = __reduce_min_sync(0xffffffffu, from), f_max = __reduce_max_sync(0xffffffffu, from);
    const int t_min = __reduce_min_sync(0xffffffffu, to), t_max = __reduce_max_sync(0xffffffffu, to);
    some = whole = 0;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      some |= (g * 16 < t_max && g * 16 + 16 > f_min ? 1u : 0u) << g;
      whole |= (g * 16 >= f_max && g * 16 + 16 <= t_min ? 1u : 0u) << g;
    }
  }
};

// What the softmax knows of a row so far: maximum (log2), R, sum of exponentials.
struct RowState {
  float m_run = -INFINITY, r_run = 0.f, l_run = 0.f;
};

// O in tensor memory for another maximum and another R.
template <int D>
__device__ __forceinline__ void rescale(uint32_t my_o, float m_new, float r_new, RowState& row) {
  const float grown = fast_exp2(row.m_run - (m_new == -INFINITY ? 0.f : m_new)), corr = grown * (r_new == row.r_run ? 1.f : page_share(row.r_run, r_new));
  row.m_run = m_new;
  row.r_run = r_new;
  row.l_run *= grown;
#pragma unroll
  for (int c = 0; c < D; c += 16) {
    uint32_t v[16];
    tmem_ld_32x32b_x16(my_o + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
    tmem_st_32x32b_x16(my_o + c, v);
  }
}

// R of a row for a tile of which it sees the columns [from, to): that of the CTA, unless it is more than 16 times the largest magnitude the row
// sees there. One that was taken once is never too large later on, since what a row has seen only grows.
__device__ __forceinline__ float row_share(int from, int to, float r_all, const float* mags, int shift, float r_run) {
  float top = 0.f;
  bool sees = false;
#pragma unroll
  for (int g = 0; g < 8; ++g)
    if (to > g * 16 && from < g * 16 + 16) {
      sees = true;
      top = fmaxf(top, mags[g >> shift]);
    }
  if (!sees) return r_run;
  return r_all == r_run || r_all <= 16.f * top ? r_all : top > r_run ? fminf(2.f * top, 3.3e38f) : r_run;
}

// One tile, as below, of rows that have an R of their own among them; 32 columns at a time, for it is not called where values are alike.
template <int D>
__device__ __noinline__ RowState softmax_apart(uint32_t my_s, uint32_t my_o, bool first, int from, int to, float row_scale, const float4* pages,
                                               const float* mags, int shift, RowState row, uint32_t p_ready) {
  const float r_new = row_share(from, to, pages[0].w, mags, shift, row.r_run);
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kT; c += 16) {
    uint32_t v[16];
    tmem_ld_32x32b_x16(my_s + c, v);
    tmem_ld_wait();
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j >= from && c + j < to) m = fmaxf(m, __uint_as_float(v[j]));
    mx = fmaxf(mx, m * (pages[c >> 4 >> shift].x * row_scale));
  }
  const float m_new = fmaxf(row.m_run, mx);
  if (first) {
    row.m_run = m_new;
    row.r_run = r_new;
  } else if (__any_sync(0xffffffffu, m_new > row.m_run + 8.f || r_new != row.r_run)) {
    rescale<D>(my_o, m_new, r_new, row);
  }
  const float m_use = row.m_run == -INFINITY ? 0.f : row.m_run, log_r = __log2f(row.r_run);
#pragma unroll 1
  for (int c = 0; c < kT; c += 32) {
    uint32_t v[32], pk[16];
    tmem_ld_32x32b_x32(my_s + c, v);  // (P takes the places of scores that have been read)
    tmem_ld_wait();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int at = ((c >> 4) + g) >> shift;
      const float scale = pages[at].x * row_scale, up = kUp + page_log(mags[at], log_r);
      float both = 0.f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        float p[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = c + g * 16 + j + k;
          p[k] = fast_exp2(fmaf(__uint_as_float(v[g * 16 + j + k]), scale, up - m_use));
          p[k] = col >= from && col < to ? p[k] : 0.f;
          both += p[k];
        }
        pk[g * 8 + (j >> 1)] = pack_f16x2(p[0], p[1]);
      }
      row.l_run += both == 0.f ? 0.f : both * fast_exp2(-up);
    }
    tmem_st_32x32b_x16(my_s + c / 2, pk);
    if (c & 32) {
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(p_ready + (c >> 6) * 8);
    }
  }
  return row;
}

// One tile of a row: S from tensor memory, P back to its place. pages: 16 bytes for each page of the tile (key magnitude / 127, log2 of its
// share of R plus kUp, the inverse of that power, R; for the second page, of which every tile has one, the smallest magnitude of values in the
// tile instead); shift: log2 of the 16-column groups in a page. INTERIOR: every column is seen, and R is the CTA's; else columns are looked
// at one by one only in the groups on an edge, and those that nobody sees cost nothing.
template <int D, bool INTERIOR>
__device__ __forceinline__ void softmax_i8(uint32_t my_s, uint32_t my_o, bool first, const Seen& seen, float row_scale, const float4* pages,
                                           const float* mags, int shift, RowState& row, uint32_t p_ready) {
  float &m_run = row.m_run, &r_run = row.r_run, &l_run = row.l_run;
  uint32_t sc[kT];
#pragma unroll
  for (int c = 0; c < kT; c += 32) tmem_ld_32x32b_x32(my_s + c, *reinterpret_cast<uint32_t(*)[32]>(&sc[c]));
  float r_new = pages[0].w;
  if constexpr (!INTERIOR) {
    bool own = false;
    if (r_new > 16.f * pages[1].w)  // (the same for all threads)
      own = r_new != r_run && (seen.to > 0 && seen.from < kT) && row_share(seen.from, seen.to, r_new, mags, shift, r_run) != r_new;
    if (__any_sync(0xffffffffu, own)) {
      tmem_ld_wait();
      row = softmax_apart<D>(my_s, my_o, first, seen.from, seen.to, row_scale, pages, mags, shift, row, p_ready);
      return;
    }
    if (!(seen.to > 0 && seen.from < kT)) r_new = r_run;  // what a row does not see leaves its R alone
  }
  tmem_ld_wait();
  float mx = -INFINITY;
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if constexpr (!INTERIOR) {
      if (!(seen.some >> g & 1)) continue;
      if (!(seen.whole >> g & 1)) {
#pragma unroll
        for (int j = g * 16; j < g * 16 + 16; ++j)
          if (j < seen.from || j >= seen.to) sc[j] = 0xff800000u;  // -inf
      }
    }
    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        m2[k] = fmaxf(fmaxf(m2[k], __uint_as_float(sc[g * 16 + j + k])), __uint_as_float(sc[g * 16 + j + 2 + k]));
    }
    mx = fmaxf(mx, fmaxf(m2[0], m2[1]) * (pages[g >> shift].x * row_scale));  // (a NaN is passed over, also -inf times 0)
  }
  const float m_new = fmaxf(m_run, mx);
  if (first) {
    m_run = m_new;
    r_run = r_new;
  } else if (__any_sync(0xffffffffu, m_new > m_run + 8.f || r_new != r_run)) {
    rescale<D>(my_o, m_new, r_new, row);
  }
  const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int c = h * 64; c < h * 64 + 64; c += 32) {
      uint32_t pk[16];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int at = (c >> 4) + g;
        if (!INTERIOR && !(seen.some >> at & 1)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pk[g * 8 + j] = 0u;
          continue;
        }
        const bool edge = !INTERIOR && !(seen.whole >> at & 1);
        const float4 page = pages[at >> shift];
        const float scale = page.x * row_scale, off = page.y - m_use;
        const uint64_t scale2 = pair2(scale, scale), off2 = pair2(off, off);
        uint64_t sum = 0ull;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float s0 = __uint_as_float(sc[c + g * 16 + j]), s1 = __uint_as_float(sc[c + g * 16 + j + 1]);
          const float2 x = unpair2(fma2(pair2(s0, s1), scale2, off2));
          float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
          if (edge) {  // (a magnitude of zero, or none, of a key that is not seen)
            p0 = s0 == -INFINITY ? 0.f : p0;
            p1 = s1 == -INFINITY ? 0.f : p1;
          }
          sum = add2(sum, pair2(p0, p1));
          pk[g * 8 + (j >> 1)] = pack_f16x2(p0, p1);
        }
        const float2 two = unpair2(sum);
        const float both = two.x + two.y;
        l_run += INTERIOR || both != 0.f ? both * page.z : 0.f;
      }
      tmem_st_32x32b_x16(my_s + c / 2, pk);
    }
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(p_ready + 8 * h);
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_i8_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sm0 = smem_u32(smem);
  float4* pages_sm = reinterpret_cast<float4*>(smem + S::kOffPages);
  float* mags_sm = reinterpret_cast<float*>(smem + S::kOffMags);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
  // q_full, q_ready | codes_full, codes_empty [kStages] | kv_full, kv_empty [kSlots] | s_full, o_full [2] | p_ready [2][2]
  const uint32_t q_full = smem_u32(bars), q_ready = q_full + 8, codes_full = q_full + 16, codes_empty = codes_full + 8 * S::kStages,
                 kv_full = codes_empty + 8 * S::kStages, kv_empty = kv_full + 8 * S::kSlots, s_full = kv_empty + 8 * S::kSlots,
                 o_full = s_full + 16, p_ready = o_full + 16;
  static_assert((2 + 2 * S::kStages + 2 * S::kSlots + 8) * 8 + 12 <= 256);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 + 2 * S::kStages + 2 * S::kSlots + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* none_flag = abort_flag + 1;  // some page's values have no magnitude
  pdl_wait();

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.x % a.Hkv, split = blockIdx.y, G = a.Hq / a.Hkv;
  const int q_begin = a.cu_q[b], L = a.cu_q[b + 1] - q_begin, ctx = a.ctx_lens[b];
  const int per_unit = kRowsQ / G;  // tokens
  // heavy blocks (late queries see the most keys) are scheduled first, of all heads (head by head: 827 us for 806)
  const int q0 = (static_cast<int>(gridDim.x) / a.Hkv - 1 - static_cast<int>(blockIdx.x) / a.Hkv) * 2 * per_unit;
  if (q0 >= L) return;  // uniform for the CTA, before any barrier or allocation
  if (q_begin < 0 || q_begin > a.T - L || L > a.max_q_len) {  // rows that are not there, or more than the grid has CTAs for
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, PXL_DEV_BAD_INDEX);
    return;
  }
  const int units = L - q0 > per_unit ? 2 : 1, tokens = min(L - q0, 2 * per_unit);
  const int pos0 = ctx - L + q0;      // position of the first token
  const int hi = pos0 + tokens;       // keys [lo, hi) are seen by some row
  const int lo = (a.window > 0 && pos0 - a.window + 1 > 0) ? pos0 - a.window + 1 : 0;
  const int t_first = lo / kT, t_all = hi > lo ? ceil_div(hi, kT) - t_first : 0, t_each = ceil_div(t_all, a.splits);
  const int t_begin = t_first + min(split * t_each, t_all);
  const int n_tiles = __shfl_sync(0xffffffffu, min(t_each, t_first + t_all - t_begin), 0);

  if (threadIdx.x == 0) {
    *abort_flag = *none_flag = 0;
    const int ppt = kT / a.page;
    mbar_init(q_full, 1);
    mbar_init(q_ready, 4 * units);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(codes_full + 8 * s, 1 + ppt);  // the bytes, and each page's numbers
      mbar_init(codes_empty + 8 * s, 4);
    }
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(kv_full + 8 * s, 4);
      mbar_init(kv_empty + 8 * s, 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(s_full + 8 * u, 1);
      mbar_init(o_full + 8 * u, 1);
      for (int h = 0; h < 2; ++h) mbar_init(p_ready + 16 * u + 8 * h, 4);  // one arrival per softmax warp of the unit
    }
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);  // S_0 | S_1 | O_0 | O_1
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_launch_dependents();
  const uint32_t tm_s = *tmem_slot, tm_o = tm_s + 2 * kT;

  // 512 threads x 128 registers at launch cover 256 x 200 + 256 x 56
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == kProducerWarp && n_tiles > 0) {
      // ------------------------------------------------------------------ TMA producer: lane p has page p of a tile
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, units * (D / 64) * per_unit * G * 128);
        for (int u = 0; u < units; ++u)
          for (int h = 0; h < D / 64; ++h)
            tma_load_3d(sm0 + u * S::kTile + h * kHalf, &tm_q, q_full, h * 64, kvh * G, q_begin + q0 + u * per_unit);
      }
      const int ppt = kT / a.page;
      const int* bt = a.block_tables + static_cast<size_t>(b) * a.max_blocks;
      auto block_of = [&](int it) {
        if (lane >= ppt || it >= n_tiles) return -1;
        int bi = (t_begin + it) * ppt + lane;
        if (bi * a.page >= ctx) bi = (ctx - 1) / a.page;  // beyond the context: the last page again (masked)
        return bi < a.max_blocks ? bt[bi] : -1;
      };
      auto head_of = [&](int blk, int it) {
        if (lane < ppt && it < n_tiles && (blk < 0 || blk >= a.num_blocks)) {
          if (a.status) atomicCAS(a.status, 0, PXL_DEV_BAD_BLOCK_PREFILL);
          blk = 0;
        }
        return (lane < ppt && it < n_tiles ? blk : 0) * a.Hkv + kvh;
      };
      int head = head_of(block_of(0), 0), blk = block_of(1);
      float2 most = a.kv_max[head];
      float r_all = 0.f;
      bool ok = true;
      int item = 0;
      for (int it = 0; ok && it < n_tiles; ++it) {
        const int next_head = head_of(blk, it + 1);
        const float2 next = a.kv_max[next_head];  // on its way while this tile is issued
        blk = block_of(it + 2);
        // the codes first; then R and the tile's pages, which the barrier of the keys counts
        for (int kv = 0; ok && kv < 2; ++kv, ++item) {
          const int stage = item % S::kStages;
          if (item >= S::kStages)
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(codes_empty + 8 * stage, (item / S::kStages - 1) & 1, abort_flag, a.status,
                                                           PXL_DEV_TIMEOUT_EMPTY));
          if (!ok) break;
          const uint32_t bar = codes_full + 8 * stage, dst = sm0 + S::kOffCodes + stage * S::kCodes + lane * a.page * D;
          if (lane == 0) mbar_arrive_expect_tx(bar, S::kCodes);
          __syncwarp();
          if (lane < ppt) {
            tma_load_2d(dst, kv ? &tm_v : &tm_k, bar, 0, head * a.page);
            if (kv == 1) mbar_arrive(bar);
          }
          if (kv == 0) {
            const int tok = (t_begin + it) * kT + lane * a.page;
            float m = lane < ppt && tok < hi && tok + a.page > lo ? most.y : 0.f;
            m = m == m ? m : 0.f;
            const float low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(m > 0.f || (lane < ppt && most.y == 0.f) ? m : INFINITY)));
            m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
            if (m > r_all) r_all = fminf(2.f * m, 3.3e38f);
            if (lane < ppt) {
              // (any share does for values without a magnitude: the sum of exponentials depends on the keys alone)
              const float share = most.y == most.y ? fmaxf(page_share(most.y, r_all), 0x1p-40f) : 1.f;
              if (most.y != most.y) *none_flag = 1;
              pages_sm[(it % kRing) * 8 + lane] = make_float4(most.x * kInv127, __log2f(share) + kUp, __fdividef(0x1p-7f, share), lane == 1 ? low : r_all);
              mags_sm[(it % kRing) * 8 + lane] = most.y;
              mbar_arrive(bar);
            }
          }
        }
        head = next_head;
        most = next;
      }
    } else if (warp == kMmaWarp && n_tiles > 0) {
      // ------------------------------------------------------------------ MMA issuer
      const uint32_t leader = elect_leader();
      auto wait = [&](uint32_t bar, int parity, int code) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, a.status, code));
        tc_fence_after_sync();
        return ok;
      };
      auto slot_of = [](int item) { return item % S::kSlots; };  // item 2 i: K of tile i, 2 i + 1: V
      auto full = [&](int item) { return wait(kv_full + 8 * slot_of(item), (item / S::kSlots) & 1, PXL_DEV_TIMEOUT_FULL); };
      auto issue_s = [&](int u, int it) {
        const uint32_t q = sm0 + u * S::kTile, k = sm0 + S::kOffKV + slot_of(2 * it) * S::kTile;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 32;
          mma_ss(tm_s + u * kT, umma_desc_k_sw128(q + off), umma_desc_k_sw128(k + off), S::kIdescS, ks > 0 ? 1u : 0u, leader);
        }
        commit(s_full + 8 * u, leader);
      };
      bool ok = wait(q_ready, 0, PXL_DEV_TIMEOUT_FULL) && full(0);
      if (ok) {
        for (int u = 0; u < units; ++u) issue_s(u, 0);
        commit(kv_empty + 8 * slot_of(0), leader);
      }
      for (int it = 0; ok && it < n_tiles; ++it) {
        const bool more = it + 1 < n_tiles;
        ok = full(2 * it + 1) && (!more || full(2 * it + 2));  // (there by now; waiting between the products would hold them up)
        const uint64_t dv = desc_v(sm0 + S::kOffKV + slot_of(2 * it + 1) * S::kTile);
        for (int u = 0; ok && u < units; ++u) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(p_ready + 16 * u + 8 * h, it & 1, PXL_DEV_TIMEOUT_TMEM_EMPTY);
            if (!ok) break;
#pragma unroll
            for (int ks = 4 * h; ks < 4 * h + 4; ++ks)  // 16 keys: 8 columns of P, 16 rows of V
              mma_ts(tm_o + u * D, tm_s + u * kT + ks * 8, dv + 128 * ks, S::kIdescPV, (it > 0 || ks > 0) ? 1u : 0u, leader);
          }
          if (!ok) break;
          if (u == units - 1) commit(kv_empty + 8 * slot_of(2 * it + 1), leader);
          if (!more) commit(o_full + 8 * u, leader);
          if (more) {
            issue_s(u, it + 1);
            if (u == units - 1) commit(kv_empty + 8 * slot_of(2 * it + 2), leader);
          }
        }
      }
    } else if (warp >= kConvertWarp) {
      // ------------------------------------------------------------------ codes -> f16 tiles
      for (int item = 0; item < 2 * n_tiles; ++item) {
        const int stage = item % S::kStages, slot = item % S::kSlots;
        bool ok = mbar_wait_bounded(codes_full + 8 * stage, (item / S::kStages) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_FULL);
        if (ok && item >= S::kSlots)
          ok = mbar_wait_bounded(kv_empty + 8 * slot, (item / S::kSlots - 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) break;
        convert_tile<D>(sm0 + S::kOffCodes + stage * S::kCodes, sm0 + S::kOffKV + slot * S::kTile, warp - kConvertWarp, lane);
        fence_proxy_async_smem();  // written through the generic proxy, read by the tensor cores through the async one
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(kv_full + 8 * slot);
          mbar_arrive(codes_empty + 8 * stage);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax warps
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int u = warp >> 2, q4 = warp & 3;
    if (u < units) {
      const int r = q4 * 32 + lane, tok = u * per_unit + r / G, head = kvh * G + r % G;  // query row = TMEM lane
      const bool valid = r < per_unit * G && tok < tokens;
      const int last = pos0 + min((u + 1) * per_unit, tokens) - 1;  // the unit's last position
      const int q_pos = min(pos0 + tok, last);                      // (rows that are nobody's: as the last)
      const int key_lo = (a.window > 0 && q_pos - a.window + 1 > 0) ? q_pos - a.window + 1 : 0;
      const uint32_t lane_sel = static_cast<uint32_t>(q4 * 32) << 16;
      const uint32_t my_s = tm_s + u * kT + lane_sel, my_o = tm_o + u * D + lane_sel;
      const int shift = a.page == 16 ? 0 : a.page == 32 ? 1 : 2;
      RowState row;
      float row_scale = 0.f;
      int failed = 0;
      if (n_tiles > 0) {
        failed = mbar_wait_bounded(q_full, 0, abort_flag, a.status, PXL_DEV_TIMEOUT_FULL) ? 0 : 1;
        if (!failed) row_scale = convert_row<D>(sm0 + u * S::kTile + r * 128, r, valid) * a.scale_log2;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
      }
      for (int it = 0; it < n_tiles; ++it) {
        const int key0 = (t_begin + it) * kT;
        const float4* pages = pages_sm + (it % kRing) * 8;
        const float* mags = mags_sm + (it % kRing) * 8;
        // every key is seen by every row of the unit, and no row has an R of its own (nor can it, unless a window hid keys before)
        bool interior = key0 + kT - 1 <= pos0 + u * per_unit && (a.window <= 0 || key0 > last - a.window);
        Seen seen;
        if (!interior) seen = Seen(key_lo - key0, q_pos + 1 - key0);
        else if (a.window > 0 && it > 0) interior = !__any_sync(0xffffffffu, row.r_run != pages_sm[((it - 1) % kRing) * 8].w);
        failed = mbar_wait_bounded(s_full + 8 * u, it & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_TMEM_FULL) ? 0 : 1;
        failed = __any_sync(0xffffffffu, failed);  // warp-uniform: the TMEM accesses below are warp-wide
        if (failed) break;
        tc_fence_after_sync();
        if (interior)
          softmax_i8<D, true>(my_s, my_o, it == 0, seen, row_scale, pages, mags, shift, row, p_ready + 16 * u);
        else
          softmax_i8<D, false>(my_s, my_o, it == 0, seen, row_scale, pages, mags, shift, row, p_ready + 16 * u);
      }
      if (!failed && n_tiles > 0) failed = mbar_wait_bounded(o_full + 8 * u, 0, abort_flag, a.status, PXL_DEV_TIMEOUT_TMEM_FULL) ? 0 : 1;
      failed = __any_sync(0xffffffffu, failed);
      bool none = false;  // the row sees values without a magnitude: its output is no number. Looked up here, and not tile by tile: a
                          // register more in the loop is a tenth of the time
      if (!failed && n_tiles > 0 && *none_flag) {
        const int end = min(q_pos, (t_begin + n_tiles) * kT - 1);
        for (int p = max(key_lo, t_begin * kT) / a.page; p < a.max_blocks && p * a.page <= end; ++p) {
          const int blk = a.block_tables[static_cast<size_t>(b) * a.max_blocks + p];
          const float m = blk >= 0 && blk < a.num_blocks ? a.kv_max[blk * a.Hkv + kvh].y : 0.f;
          none = none || m != m;
        }
      }
      const auto [m_run, r_run, l_run] = row;
      const int64_t place = static_cast<int64_t>(q_begin + q0 + tok) * a.Hq + head;
      if (!failed && a.splits == 1) {
        const float sink = a.sinks && valid ? a.sinks[head] * kLog2e : -INFINITY;
        const float M = fmaxf(m_run, sink), Mu = M == -INFINITY ? 0.f : M, f = fast_exp2(m_run - Mu);
        const float denom = l_run * f + fast_exp2(sink - Mu);
        if (a.lse && valid) a.lse[place] = denom == 0.f ? INFINITY : Mu + log2f(denom);
        const float inv = none ? NAN : denom == 0.f ? 0.f : f / denom * (r_run * (kInv127 * 0x1p-7f));
        bf16* dst = a.out + static_cast<int64_t>(q_begin + q0 + tok) * a.out_stride + head * D;
        if (n_tiles > 0) tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          if (n_tiles > 0) {
            tmem_ld_32x32b_x32(my_o + c, v);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          }
#pragma unroll
          for (int c8 = 0; c8 < 32; c8 += 8) {
            bf16x8 ov;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              ov.u[j] = denom == 0.f ? 0u
                                     : pack_bf16x2(__uint_as_float(v[c8 + 2 * j]) * inv, __uint_as_float(v[c8 + 2 * j + 1]) * inv);
            if (valid) st_bf16x8(dst + c + c8, ov);
          }
        }
      } else if (!failed) {
        float* po = a.parts + (split * static_cast<int64_t>(a.T) * a.Hq + place) * (D + kPartTail);
        if (valid) *reinterpret_cast<float4*>(po + D) = make_float4(m_run, l_run, r_run, none ? 1.f : 0.f);
        if (n_tiles > 0) {
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(my_o + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              if (valid) *reinterpret_cast<uint4*>(po + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
      }
      tc_fence_before_sync();
    }
  }

  // ---------------------------------------------------------------------- teardown
  __syncwarp();
  if (*abort_flag) __nanosleep(200000);  // loads that are still in flight must land before smem is released
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == kMmaWarp) tmem_dealloc(tm_s, 512);
}

// Adds up the parts of a row of a split call: a warp per (token, query head).
template <int D>
__global__ void __launch_bounds__(128)
attn_i8_prefill_join_kernel(const __grid_constant__ Args a, int B) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5), rows = static_cast<int64_t>(a.T) * a.Hq;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int token = static_cast<int>(row / a.Hq), head = static_cast<int>(row % a.Hq);
  bool there = false;  // in a sequence that has parts; one that was reported has none
  if (row < rows)
    for (int b = lane; b < B; b += 32) {
      const int begin = a.cu_q[b], end = a.cu_q[b + 1];
      there = there || (begin >= 0 && end <= a.T && end - begin <= a.max_q_len && token >= begin && token < end);
    }
  if (!__any_sync(0xffffffffu, there)) return;
  const float sink = a.sinks ? a.sinks[head] * kLog2e : -INFINITY;
  const float* p = a.parts + row * (D + kPartTail);
  const int64_t next = rows * (D + kPartTail);
  float M = -INFINITY, R = 0.f;
  bool none = false;
  for (int s = lane; s < a.splits; s += 32) {
    const float4 t = *reinterpret_cast<const float4*>(p + s * next + D);
    none = none || t.w != 0.f;
    M = fmaxf(M, t.x);
    R = fmaxf(R, t.z);
  }
  M = warp_reduce_max(M);
  R = warp_reduce_max(R);
  const float top = fmaxf(M, sink), Mu = top == -INFINITY ? 0.f : top;
  float l = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int s0 = 0; s0 < a.splits; s0 += 32) {
    float f = 0.f;  // of part s0 + lane; 0 where none of its keys is seen (and its output was not written)
    bool some = false;
    if (s0 + lane < a.splits) {
      const float4 t = *reinterpret_cast<const float4*>(p + (s0 + lane) * next + D);
      some = t.y != 0.f;
      f = some ? fast_exp2(t.x - Mu) : 0.f;
      l += some ? t.y * f : 0.f;
      f *= page_share(t.z, R);
    }
    const uint32_t written = __ballot_sync(0xffffffffu, some);
    const int n = min(32, a.splits - s0);
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float fs = __shfl_sync(0xffffffffu, f, s);
      const bool in = written >> s & 1;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const float o = in ? p[(s0 + s) * next + i * 32 + lane] : 0.f;
        acc[i] += in ? o * fs : 0.f;
      }
    }
  }
  l = warp_reduce_sum(l) + fast_exp2(sink - Mu);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? INFINITY : Mu + log2f(l);
  const float inv = __any_sync(0xffffffffu, none) ? NAN : l == 0.f ? 0.f : R * (kInv127 * 0x1p-7f) / l;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) a.out[token * a.out_stride + head * D + i * 32 + lane] = __float2bfloat16(acc[i] * inv);
}

// CTAs that share a block of queries' keys: as many as fill the chip, each with at least four tiles.
int splits_of(int B, int max_q_len, int Hq, int Hkv, int max_ctx) {
  const int64_t blocks = static_cast<int64_t>(ceil_div(max_q_len > 0 ? max_q_len : 1, 2 * (kRowsQ / (Hq / Hkv)))) * Hkv * B;
  const int64_t fill = pxl_host::num_sms() / (blocks > 0 ? blocks : 1), most = max_ctx / (4 * kT);
  const int64_t s = fill < most ? fill : most;
  return s < 1 ? 1 : static_cast<int>(s);
}

struct Layout {  // floats of the workspace
  int splits;
  int64_t total;
  Layout(int T, int B, int max_q_len, int Hq, int Hkv, int D, int max_ctx) {
    splits = splits_of(B, max_q_len, Hq, Hkv, max_ctx);
    const int64_t rows = static_cast<int64_t>(T) * Hq;
    total = splits > 1 ? splits * rows * (D + kPartTail) : 0;
  }
};

template <int D>
int launch_prefill(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int B, int max_q_len, cudaStream_t stream) {
  static std::atomic<bool> configured[64];  // function attributes are per device
  std::atomic<bool>& done = configured[pxl_host::current_device_slot()];
  if (!done.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(attn_i8_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem) != cudaSuccess)
      return PXL_ERR_CUDA;
    done.store(true, std::memory_order_relaxed);
  }
  const int blocks = ceil_div(max_q_len > 0 ? max_q_len : 1, 2 * (kRowsQ / (a.Hq / a.Hkv)));
  if (static_cast<int64_t>(blocks) * a.Hkv > INT32_MAX || a.splits > 65535) return PXL_ERR_TOO_LARGE;
  pxl_host::launch(attn_i8_prefill_kernel<D>, dim3(blocks * a.Hkv, a.splits, B), dim3(kThreads), Shape<D>::kSmem, stream, tq, tk, tv, a);
  if (a.splits > 1)
    pxl_host::launch_behind(attn_i8_prefill_join_kernel<D>, dim3(static_cast<unsigned>(ceil_div64(static_cast<int64_t>(a.T) * a.Hq, 4))), dim3(128),
                            0, stream, a, B);
  return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

}  // namespace

PXL_EXPORT int64_t pxl_attn_i8_prefill_workspace(int T, int B, int max_q_len, int Hq, int Hkv, int D, int max_ctx) {
  if (T <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || max_q_len < 0) return 0;
  return Layout(T, B, max_q_len, Hq, Hkv, D, max_ctx).total * 4;
}

PXL_EXPORT int pxl_attn_i8_prefill(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const float* kv_max,
                                   const int* block_tables, const int* cu_q, const int* ctx_lens, void* out, int64_t out_stride,
                                   const float* sinks, float* lse, void* workspace, int64_t workspace_bytes, int T, int B, int max_q_len,
                                   int Hq, int Hkv, int D, int page, int max_blocks, int64_t num_blocks, float scale, int window, int max_ctx,
                                   int* status, cudaStream_t stream) {
  if (T <= 0 || B <= 0) return PXL_OK;
  if ((D != 64 && D != 128) || (page != 16 && page != 32 && page != 64) || Hkv <= 0 || Hq % Hkv || Hq / Hkv < 1 || Hq / Hkv > 16 ||
      !(scale > 0.f) || (q_stride & 7) || (out_stride & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (reinterpret_cast<uintptr_t>(kv_max) & 7) || max_blocks <= 0 || max_q_len < 0 || max_ctx <= 0 || max_ctx >= (1 << 30) ||
      window < 0 || window > (1 << 30) || num_blocks <= 0 ||
      num_blocks * Hkv * page >= (1ll << 31))
    return PXL_ERR_INVALID_ARG;
  const Layout at(T, B, max_q_len, Hq, Hkv, D, max_ctx);
  if (workspace_bytes < at.total * 4 || (at.total > 0 && !workspace)) return PXL_ERR_INVALID_ARG;
  if (B > 65535) return PXL_ERR_TOO_LARGE;
  CUtensorMap tq, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * Hkv * page;
  if (!pxl_host::make_tmap_queries(&tq, q, q_stride, T, Hq, D, Hq / Hkv) || !pxl_host::make_tmap_codes(&tk, k_cache, rows, D, page) ||
      !pxl_host::make_tmap_codes(&tv, v_cache, rows, D, page))
    return PXL_ERR_TENSORMAP;
  const Args a{reinterpret_cast<const float2*>(kv_max), block_tables, cu_q, ctx_lens, static_cast<bf16*>(out), out_stride, sinks, lse,
               static_cast<float*>(workspace), T, max_q_len, Hq, Hkv, page, max_blocks, num_blocks, scale * kLog2e, window, at.splits, status};
  return D == 64 ? launch_prefill<64>(tq, tk, tv, a, B, max_q_len, stream) : launch_prefill<128>(tq, tk, tv, a, B, max_q_len, stream);
}
