// Keys and values in 8 bits: writing new tokens into such a cache, reading sequences out of it, thinning them out.
//
// A cache holds pages [blocks, Hkv, page, D] of int8 codes for K and as many for V, and kv_max fp32 [blocks, Hkv, 2]: the largest
// magnitude m of a page's keys and of its values. A code c stands for c * (m / 127). Codes are round(127 x / m), ties to even: 127 x is
// exact in fp32 for bf16 x, and m is a bf16 number too. With x / m = X / (M 2^k), X and M whole numbers of 8 bits, the quotient is off a
// tie j / 2 by |254 X - j M 2^k| / (2 M 2^k): not at all, or by at least 1 / (254 X + 1) > 2^-16 of the tie (16383 / 32768 for
// x = 129 / 32768 and m = 1). The rounded quotient is off by 2^-24 of itself and gives the code of the exact one. Tokens behind a page's
// first may raise m; the codes that are there become round(c * m_old / m_new), also from an exact product and as far from ties. m is NaN
// once a page was given a number that is not finite, until its first token is written again. (Magnitudes of a caller's own that are no
// bf16 numbers do as well, but for codes that are written again from within 2^-16 of a tie, which may be the neighbour of the nearest.)
#include <atomic>

#include "common.cuh"
#include "kv_i8.cuh"
#include "pxl_api.h"

namespace {
using namespace pxl;

// Quotients p / m of four numbers, p exact, as correctly rounded fp32 (Markstein: one correction of p * (1 / m) by its remainder, which a
// fused multiply-add has exactly), then to the nearest integer, ties to even, as bytes: 2.5 operations a number on register pairs, no
// branch. (A division each is ten times that, and was most of these kernels' time.) m scaled into [1, 2), p alike.
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: a number below 2^22 that is added to it is rounded to an integer, its low bits
struct Divider {
  float inv;
  uint64_t inv2, neg2;
  // `unit`: the power of two that p is to be multiplied by
  __device__ __forceinline__ Divider(float m, float& unit) {
    const int e = static_cast<int>(__float_as_uint(m) >> 23);  // of m below 2^-100: that of 2^-100
    unit = __uint_as_float(static_cast<uint32_t>(e < 27 ? 227 : e > 253 ? 1 : 254 - e) << 23);
    const float scaled = m * unit;
    inv = m > 0.f ? __frcp_rn(scaled) : 0.f;
    inv2 = pair2(inv, inv);
    neg2 = pair2(-scaled, -scaled);
  }
  __device__ __forceinline__ uint32_t operator()(uint64_t p01, uint64_t p23) const {
    uint64_t n[2];
    const uint64_t p[2] = {p01, p23}, magic = pair2(kMagic, kMagic);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t q = mul2(p[i], inv2);
      n[i] = add2(fma2(fma2(q, neg2, p[i]), inv2, q), magic);
    }
    const float2 a = unpair2(n[0]), b = unpair2(n[1]);
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040),
                       0x5410);
  }
};

// round(127 x / m) of four numbers; 0 for a page of zeros or without a magnitude
struct Coder {
  float unit;
  Divider by;
  bool none;
  __device__ __forceinline__ explicit Coder(float m) : unit(0.f), by(m, unit), none(!(m > 0.f)) { unit *= 127.f; }
  __device__ __forceinline__ uint32_t operator()(float2 a, float2 b) const {
    if (none) return 0;
    const uint64_t up = pair2(unit, unit);
    return by(mul2(pair2(a.x, a.y), up), mul2(pair2(b.x, b.y), up));
  }
};

// the numbers of bytes I and I + 1 of a word of codes with their sign bits flipped: under the exponent of 2^23
template <int I>
__device__ __forceinline__ uint64_t codes_f32x2(uint32_t flipped) {
  const uint32_t a = __byte_perm(flipped, 0x4b000000u, 0x7440 + I), b = __byte_perm(flipped, 0x4b000000u, 0x7441 + I);
  return add2(pair2(__uint_as_float(a), __uint_as_float(b)), pair2(-8388736.f, -8388736.f));
}

// round(c * from / to); as it is where the new magnitude is no number
struct Recoder {
  float to, unit;
  Divider by;
  __device__ __forceinline__ explicit Recoder(float to) : to(to), unit(0.f), by(to, unit) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t four, float from) const {
    if (from == to || !(to == to)) return four;
    const uint32_t f = flip_codes(four);
    const uint64_t up = pair2(from * unit, from * unit);
    return by(mul2(codes_f32x2<0>(f), up), mul2(codes_f32x2<2>(f), up));
  }
};

// x / 127, correctly rounded
__device__ __forceinline__ float over_127(float x) {
  if (!(fabsf(x) > 0x1p-100f)) return __fdiv_rn(x, 127.f);
  const float q = x * (1.f / 127.f);
  return fmaf(fmaf(-127.f, q, x), 1.f / 127.f, q);
}

// ---- write ---------------------------------------------------------------------------------------------------------
// One CTA per (page that gets tokens, key head): HALF threads for the keys and as many for the values, which keep what they read. ROWS: new
// tokens that a page gets at most (1 in a decoding step, with a warp for each half). 12000 tokens of 8 heads in prompts 19 us, 2.6 TB/s in and
// out: load, meet, round and store follow one another in a CTA. (Four CTAs on an SM for pages of 64: 21 -> 19.)
template <int D, int ROWS, int HALF>
__global__ void __launch_bounds__(2 * HALF, D == 128 && ROWS == 64 ? 4 : 0)
store_kv_i8_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t k_stride, int64_t v_stride,
                   const int* __restrict__ block_tables, const int* __restrict__ cu_q, const int* __restrict__ ctx_lens,
                   int8_t* __restrict__ k_cache, int8_t* __restrict__ v_cache, float* __restrict__ kv_max, int T, int max_q_len, int Hkv,
                   int page, int max_blocks, int64_t num_blocks, int* status) {
  constexpr int C = D / 8, kSteps = ceil_div(ROWS * C, HALF);  // chunks of 8 values in a row; of a thread
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, kv = threadIdx.x / HALF, tid = threadIdx.x % HALF;
  const int row0 = cu_q[b], n = cu_q[b + 1] - row0, t = ctx_lens[b];
  const int begin = t - n, from = begin > 0 ? begin : 0;
  const int p = from / page + static_cast<int>(blockIdx.x);
  if (n > max_q_len) {  // the grid has no CTAs for all its pages: none of them
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_INDEX);
    return;
  }
  if (n <= 0 || t <= 0 || p > (t - 1) / page) return;
  const int lo = from > p * page ? from - p * page : 0, hi = min(page, t - p * page), rows = hi - lo;
  const int first = row0 + p * page + lo - begin;  // row of token lo of the page
  const int blk = p < max_blocks ? block_tables[static_cast<size_t>(b) * max_blocks + p] : -1;
  const bool fits = first >= 0 && first + rows <= T && rows <= ROWS;
  const int64_t stride = kv ? v_stride : k_stride;
  const bf16* src = (kv ? v : k) + static_cast<int64_t>(first) * stride + h * D;
  bf16x8 x[kSteps];  // (on their way while the block is looked up)
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = s * HALF + tid;
    if (fits && i < rows * C) x[s] = ld_bf16x8(src + (i / C) * stride + (i % C) * 8);
  }
  if (blk < 0 || blk >= num_blocks || !fits) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
    return;
  }
  int8_t* dst = (kv ? v_cache : k_cache) + (static_cast<size_t>(blk) * Hkv + h) * page * D;
  float* m_at = kv_max + (static_cast<size_t>(blk) * Hkv + h) * 2 + kv;

  const float old = lo > 0 ? *m_at : 0.f;
  uint32_t top = 0;  // bits of the largest magnitude: ordered like the numbers, infinities and NaN above all of them
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (s * HALF + tid >= rows * C) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, max(x[s].u[j] & 0x7fffu, (x[s].u[j] >> 16) & 0x7fffu));
  }
  __shared__ uint32_t tops[2 * HALF / 32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < HALF / 32; ++w) top = max(top, tops[kv * (HALF / 32) + w]);
  const float now = top >= 0x7f80u || !(old == old) ? __uint_as_float(0x7fc00000u) : fmaxf(old, __uint_as_float(top << 16));
  if (tid == 0) *m_at = now;
  if (lo > 0 && now > old) {
    const Recoder again(now);
    for (int i = tid; i < lo * C; i += HALF) {
      const uint2 c = *reinterpret_cast<const uint2*>(dst + i * 8);
      *reinterpret_cast<uint2*>(dst + i * 8) = make_uint2(again(c.x, old), again(c.y, old));
    }
  }
  const Coder code(now);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = s * HALF + tid;
    if (i >= rows * C) break;
    *reinterpret_cast<uint2*>(dst + lo * D + i * 8) = make_uint2(code(unpack_bf16x2(x[s].u[0]), unpack_bf16x2(x[s].u[1])),
                                                                code(unpack_bf16x2(x[s].u[2]), unpack_bf16x2(x[s].u[3])));
  }
}

// ---- read ----------------------------------------------------------------------------------------------------------
// A warp takes a row of the result, all heads, keys and values: it finds the row's sequence by counting the ends at or before it, then has 8
// codes per lane of keys and of values in four steps in flight, and its stores are whole lines. 82000 tokens of 8 heads 88 us, 5.0 TB/s. (16 rows
// to a CTA, found by bisection, one load behind the other: 105 us; two rows to a warp 100; five CTAs on an SM 92.)
constexpr int kLoadWarps = 8;
template <int D>
__global__ void __launch_bounds__(kLoadWarps * 32, 6)
load_kv_i8_kernel(const int8_t* __restrict__ k_cache, const int8_t* __restrict__ v_cache, const float* __restrict__ kv_max,
                  const int* __restrict__ block_tables, const int* __restrict__ cu_k, bf16* __restrict__ k_out, bf16* __restrict__ v_out, int rows,
                  int B, int Hkv, int page, int max_blocks, int64_t num_blocks, int* status) {
  constexpr int C = D / 8, kHeads = 32 / C, kFlight = 4;  // heads of a step
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * kLoadWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  int before = 0, begin = 0;  // sequences that begin at or before the row; where the last of these does
  for (int i = lane; i <= B; i += 32) {
    const int at = cu_k[i];
    if (at <= row) ++before, begin = max(begin, at);
  }
  before = __reduce_add_sync(0xffffffffu, before);
  begin = __reduce_max_sync(0xffffffffu, begin);
  int blk = -1, off = 0;
  if (before > 0 && before <= B) {
    const int p = (row - begin) / page;
    blk = p < max_blocks ? block_tables[static_cast<size_t>(before - 1) * max_blocks + p] : -1;
    off = (row - begin) % page;
    if (blk < 0 || blk >= num_blocks) {
      if (lane == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
      blk = -1;
    }
  }
  const size_t src = (static_cast<size_t>(blk < 0 ? 0 : blk) * Hkv * page + off) * D + lane % C * 8;
  const float2* most = reinterpret_cast<const float2*>(kv_max) + static_cast<size_t>(blk < 0 ? 0 : blk) * Hkv;
  const size_t dst = static_cast<size_t>(row) * Hkv * D + lane % C * 8;
  for (int h0 = lane / C; h0 < Hkv; h0 += kHeads * kFlight) {
    uint2 x[2][kFlight];
    float2 m[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const int h = h0 + j * kHeads;
      const bool in = blk >= 0 && h < Hkv;
      m[j] = in ? most[h] : make_float2(0.f, 0.f);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        x[kv][j] = in ? *reinterpret_cast<const uint2*>((kv ? v_cache : k_cache) + src + static_cast<size_t>(h) * page * D) : make_uint2(0, 0);
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const int h = h0 + j * kHeads;
      if (h >= Hkv) break;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float f = over_127(kv ? m[j].y : m[j].x);
        const uint64_t f2 = pair2(f, f);
        const uint32_t a = flip_codes(x[kv][j].x), b = flip_codes(x[kv][j].y);
        const float2 v[4] = {unpair2(mul2(codes_f32x2<0>(a), f2)), unpair2(mul2(codes_f32x2<2>(a), f2)), unpair2(mul2(codes_f32x2<0>(b), f2)),
                             unpair2(mul2(codes_f32x2<2>(b), f2))};
        bf16x8 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o.u[i] = pack_bf16x2(v[i].x, v[i].y);
        st_bf16x8((kv ? v_out : k_out) + dst + h * D, o);
      }
    }
  }
}

// ---- thin out ------------------------------------------------------------------------------------------------------
// Which tokens stay. One CTA per (sequence, key head): the weight that the last of the chosen tokens has, by its bits from the top (11,
// 11 and 10 of them, a histogram each), then the tokens above it and the earliest of those that have it, in order: each warp counts and
// then writes those of its own stretch. The weights are read from memory once and kept as keys in shared memory (CACHED: up to 50000
// tokens), or read in each of the five passes. They move to their new places chunk by chunk, the first chunk first: a token never moves
// back, so that no chunk writes where a later one reads. 40 sequences of up to 9000 tokens, 8 heads: 24 us.
constexpr int kPickThreads = 1024;
constexpr int kBins = 2048;
constexpr int kPickCache = 50000;

__device__ __forceinline__ uint32_t weight_key(float w) {  // ordered like the weights; NaN above all
  if (!(w == w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 is 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <bool CACHED>
__global__ void __launch_bounds__(kPickThreads)
evict_pick_kernel(float* __restrict__ weights, int64_t W, int slots, const int* __restrict__ seq_slots, const int* __restrict__ ctx_lens,
                  int* __restrict__ kept, int* __restrict__ new_lens, int Hkv, int capacity, int keep, int recent, int first, int* status) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t sums[32], base_above[32], base_equal[32], found[2];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = seq_slots ? seq_slots[b] : b;
  int n = max(ctx_lens[b], 0);
  bool twice = false;  // another sequence has the slot
  if (seq_slots)
    for (int i = threadIdx.x; i < static_cast<int>(gridDim.y); i += kPickThreads)
      twice = twice || (i != b && seq_slots[i] == slot && n > 0 && ctx_lens[i] > 0);
  if (__syncthreads_or(twice)) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
    n = 0;
  }
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
  auto key_of = [&](int i) { return CACHED ? keys[i] : weight_key(w[first + i]); };
  if (want > 0) {
    if (CACHED) {
#pragma unroll 8
      for (int i = threadIdx.x; i < count; i += kPickThreads) keys[i] = weight_key(w[first + i]);  // (each thread reads its own again)
    }
    uint32_t prefix = 0, left = want;  // `left` of the keys that begin with `prefix` are chosen
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t above = pass == 0 ? 0 : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = threadIdx.x; i < kBins; i += kPickThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = threadIdx.x; i < count; i += kPickThreads) {
        const uint32_t key = key_of(i);
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
#pragma unroll 4
    for (int i = lo + lane; i < hi; i += 32) {
      const uint32_t key = key_of(i);
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
#pragma unroll 4
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t key = i < hi ? key_of(i) : 0u;
      const uint32_t eq = __ballot_sync(0xffffffffu, i < hi && key == prefix), below = (1u << lane) - 1;
      const bool take = i < hi && (key > prefix || (key == prefix && ties + __popc(eq & below) < left));
      const uint32_t all = __ballot_sync(0xffffffffu, take);
      const int place = at + __popc(all & below);
      if (take && place < want) out[first + place] = first + i;  // (they are `want`, unless the weights change meanwhile)
      at += __popc(all);
      ties += __popc(eq);
    }
  }
  __syncthreads();
  constexpr int kMove = 4;
  for (int i0 = 0; i0 < keep; i0 += kMove * kPickThreads) {
    float x[kMove];
#pragma unroll
    for (int j = 0; j < kMove; ++j) {
      const int i = i0 + j * kPickThreads + threadIdx.x;
      x[j] = i < keep ? w[min(max(out[i], 0), n - 1)] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMove; ++j) {
      const int i = i0 + j * kPickThreads + threadIdx.x;
      if (i < keep) w[i] = x[j];
    }
    __syncthreads();
  }
  for (int i = keep + threadIdx.x; i < n; i += kPickThreads) w[i] = 0.f;
}

// The tokens that stay into their new pages: a warp takes 16 of a key head, with all their codes in flight (16 of them to a load). The new
// magnitude of a page is the largest that a token of it had: a warp looks all of its page's tokens up. 40 x 2048 tokens of 8 heads 88 us, 3.4
// TB/s: single rows of 128 bytes and 2.5 operations per code; eight CTAs on an SM for heads of 128: 92. (CTAs of 64 tokens that met between
// the look-up, three loads one behind the other, and the codes: 125 us.)
constexpr int kMoveWarps = 4;
template <int D, int PAGE>
__global__ void __launch_bounds__(kMoveWarps * 32, D == 128 ? 9 : 0)
evict_move_kernel(int8_t* __restrict__ k_cache, int8_t* __restrict__ v_cache, float* __restrict__ kv_max, const int* __restrict__ block_tables,
                  const int* __restrict__ new_tables, const int* __restrict__ kept, const int* __restrict__ new_lens, int Hkv, int max_blocks,
                  int max_new, int64_t num_blocks, int keep, int* status) {
  constexpr int C = D / 16, kPerStep = 32 / (2 * C), kSteps = 16 / kPerStep;  // tokens of a step: 2 C lanes each
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  const int r0 = (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * 16, n = new_lens[b];
  if (r0 >= n) return;
  const int* of = kept + (static_cast<int64_t>(b) * Hkv + h) * keep;
  const int* bt = block_tables + static_cast<size_t>(b) * max_blocks;
  auto look = [&](int r, float2& m) {  // row of token r of those that stay, in the cache; -1 for none
    m = make_float2(0.f, 0.f);
    if (r >= n) return -1;
    const int i = of[r], blk = i >= 0 && i / PAGE < max_blocks ? bt[i / PAGE] : -1;
    if (blk < 0 || blk >= num_blocks) {
      if (status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
      return -1;
    }
    m = *reinterpret_cast<const float2*>(kv_max + (static_cast<size_t>(blk) * Hkv + h) * 2);
    return (blk * Hkv + h) * PAGE + i % PAGE;  // (below 2^31: the host has checked)
  };
  const int p = r0 / PAGE, blk = p < max_new ? new_tables[static_cast<size_t>(b) * max_new + p] : -1;
  float2 m;
  const int row = look(r0 + (lane & 15), m);
  if (blk < 0 || blk >= num_blocks) {
    if (lane == 0 && status) atomicCAS(status, 0, PXL_DEV_BAD_SLOT);
    return;
  }
  const int kv = lane / C & 1, c = lane % C;
  int8_t* cache = kv ? v_cache : k_cache;
  uint4 x[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int at = __shfl_sync(0xffffffffu, row, s * kPerStep + lane / (2 * C));
    x[s] = at >= 0 ? *reinterpret_cast<const uint4*>(cache + static_cast<size_t>(at) * D + c * 16) : make_uint4(0, 0, 0, 0);
  }
  float top[2] = {m.x, m.y};
  bool none[2] = {!(m.x == m.x), !(m.y == m.y)};
  if (PAGE > 16) {
    for (int r = p * PAGE + lane; r < (p + 1) * PAGE; r += 32) {
      float2 other;
      look(r, other);
      top[0] = fmaxf(top[0], other.x), top[1] = fmaxf(top[1], other.y);  // (which pass over NaN)
      none[0] = none[0] || !(other.x == other.x), none[1] = none[1] || !(other.y == other.y);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    top[j] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(none[j] ? 0.f : top[j])));  // (none is below zero)
    if (__any_sync(0xffffffffu, none[j])) top[j] = __uint_as_float(0x7fc00000u);
  }
  const Recoder again(kv ? top[1] : top[0]);
  const size_t dst = static_cast<size_t>(blk) * Hkv + h;
  if (r0 % PAGE == 0 && lane < 2) kv_max[dst * 2 + lane] = lane ? top[1] : top[0];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int at = s * kPerStep + lane / (2 * C);
    const float mk = __shfl_sync(0xffffffffu, m.x, at), mv = __shfl_sync(0xffffffffu, m.y, at);
    const bool there = __shfl_sync(0xffffffffu, row, at) >= 0;
    const float from = kv ? mv : mk;
    const uint4 w = make_uint4(again(x[s].x, from), again(x[s].y, from), again(x[s].z, from), again(x[s].w, from));
    if (there) *reinterpret_cast<uint4*>(cache + (dst * PAGE + (r0 + at) % PAGE) * D + c * 16) = w;
  }
}

bool cache_ok(int Hkv, int D, int page, int max_blocks, int64_t num_blocks, const void* k_cache, const void* v_cache) {
  return Hkv > 0 && (D == 64 || D == 128) && (page == 16 || page == 32 || page == 64) && max_blocks > 0 && num_blocks > 0 &&
         num_blocks * Hkv * page < (1ll << 31) && !((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15);
}
bool pairs_ok(const float* kv_max) { return !(reinterpret_cast<uintptr_t>(kv_max) & 7); }  // (where they are read as such)
int done() { return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA; }

}  // namespace

PXL_EXPORT int pxl_kv_i8_store(const void* k, const void* v, int64_t k_stride, int64_t v_stride, const int* block_tables, const int* cu_q,
                               const int* ctx_lens, void* k_cache, void* v_cache, float* kv_max, int T, int B, int max_q_len, int Hkv, int D,
                               int page, int max_blocks, int64_t num_blocks, int* status, cudaStream_t stream) {
  if (B <= 0 || T <= 0) return PXL_OK;
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || max_q_len < 0 || Hkv > 65535 || (k_stride & 7) || (v_stride & 7) ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
    return PXL_ERR_INVALID_ARG;
  if (B > 65535) return PXL_ERR_TOO_LARGE;
  const dim3 grid((max_q_len + page - 2) / page + 1, Hkv, B);
  auto go = [&](auto kernel, int threads) {
    pxl_host::launch(kernel, grid, dim3(threads), 0, stream, static_cast<const bf16*>(k), static_cast<const bf16*>(v), k_stride, v_stride,
                     block_tables, cu_q, ctx_lens, static_cast<int8_t*>(k_cache), static_cast<int8_t*>(v_cache), kv_max, T, max_q_len, Hkv,
                     page, max_blocks, num_blocks, status);
    return done();
  };
  if (max_q_len <= 1) return D == 64 ? go(store_kv_i8_kernel<64, 1, 32>, 64) : go(store_kv_i8_kernel<128, 1, 32>, 64);
  if (D == 64)
    return page == 16   ? go(store_kv_i8_kernel<64, 16, 64>, 128)
           : page == 32 ? go(store_kv_i8_kernel<64, 32, 128>, 256)
                        : go(store_kv_i8_kernel<64, 64, 128>, 256);
  return page == 16   ? go(store_kv_i8_kernel<128, 16, 64>, 128)
         : page == 32 ? go(store_kv_i8_kernel<128, 32, 128>, 256)
                      : go(store_kv_i8_kernel<128, 64, 128>, 256);
}

PXL_EXPORT int pxl_kv_i8_load(const void* k_cache, const void* v_cache, const float* kv_max, const int* block_tables, const int* cu_k, void* k,
                              void* v, int rows, int B, int Hkv, int D, int page, int max_blocks, int64_t num_blocks, int* status,
                              cudaStream_t stream) {
  if (rows <= 0) return PXL_OK;
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || !pairs_ok(kv_max) || B < 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
    return PXL_ERR_INVALID_ARG;
  auto go = [&](auto kernel) {
    pxl_host::launch(kernel, dim3(ceil_div(rows, kLoadWarps)), dim3(kLoadWarps * 32), 0, stream, static_cast<const int8_t*>(k_cache),
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
  if (!cache_ok(Hkv, D, page, max_blocks, num_blocks, k_cache, v_cache) || !pairs_ok(kv_max) || max_new <= 0 || W <= 0 || keep < 1 || recent < 0 || first < 0 ||
      static_cast<int64_t>(recent) + first > keep || keep > static_cast<int64_t>(max_new) * page || static_cast<int64_t>(max_blocks) * page > INT32_MAX)
    return PXL_ERR_INVALID_ARG;
  if (B > 65535 || Hkv > 65535) return PXL_ERR_TOO_LARGE;
  const int64_t longest = W < static_cast<int64_t>(max_blocks) * page ? W : static_cast<int64_t>(max_blocks) * page;
  const bool cached = longest <= kPickCache;
  static std::atomic<bool> configured[64];  // function attributes are per device
  std::atomic<bool>& set = configured[pxl_host::current_device_slot()];
  if (!set.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(evict_pick_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickCache * 4) != cudaSuccess)
      return PXL_ERR_CUDA;
    set.store(true, std::memory_order_relaxed);
  }
  pxl_host::launch(cached ? evict_pick_kernel<true> : evict_pick_kernel<false>, dim3(Hkv, B), dim3(kPickThreads), cached ? longest * 4 : 0,
                   stream, weights, W, slots, seq_slots, ctx_lens, kept, new_lens, Hkv, max_blocks * page, keep, recent, first, status);
  if (const int rc = done()) return rc;
  auto go = [&](auto kernel) {
    pxl_host::launch_behind(kernel, dim3(ceil_div(keep, 16 * kMoveWarps), Hkv, B), dim3(kMoveWarps * 32), 0, stream, static_cast<int8_t*>(k_cache),
                     static_cast<int8_t*>(v_cache), kv_max, block_tables, new_tables, kept, new_lens, Hkv, max_blocks, max_new, num_blocks,
                     keep, status);
    pxl_host::next_launch_follows_whole();  // the new lengths
    return done();
  };
  if (D == 64) return page == 16 ? go(evict_move_kernel<64, 16>) : page == 32 ? go(evict_move_kernel<64, 32>) : go(evict_move_kernel<64, 64>);
  return page == 16 ? go(evict_move_kernel<128, 16>) : page == 32 ? go(evict_move_kernel<128, 32>) : go(evict_move_kernel<128, 64>);
}
