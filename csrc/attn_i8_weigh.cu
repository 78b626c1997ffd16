// What the queries of new tokens gave to each token of a cache in 8 bits (layout: kv_i8.cu): weights[slot, head, token] += the sum over the
// queries that see it, and over the query heads of its key head, of exp(score - log of the query's sum), on the 5th-generation tensor cores.
//
// A CTA has 256 keys of a key head, as two A operands: a key is a lane of tensor memory, and its sum stays in one thread's register, with no
// exchange between threads. Its codes become bf16 once (exactly), times the power of two in its page's magnitude and the softmax scale, so that
// the products are of the scores' size whatever that of the queries; these stream through as they are, 128 / G tokens of G heads at a time:
//   warp 16   : TMA producer, a ring of query boxes, and their rows' logarithms beside them
//   warp 17   : MMA issuer, S = K Q^T into two TMEM buffers of 128 columns for each 128 keys
//   warps 0-15: four groups of four, each with a buffer of its own: 128 exponentials per key and unit, 16 columns at a time with the next
//               scores and logarithms on their way
// 2048 tokens of 40 heads behind 14000, us: 128 keys per CTA and two groups 598; with the next 32 columns on their way 550; 256 keys per CTA,
// which halves the queries' way through L2, and four groups 484 (391 without the exponentials).
// The bound is the exponentials: 256 x 128 per unit at 16 a clock, 2048 clocks, beside 1024 of the products (D = 128).
// Long units for few keys are split over CTAs, whose sums a second kernel adds in their order.
#include <atomic>

#include "attention_rows.cuh"
#include "common.cuh"
#include "kv_i8.cuh"
#include "pxl_api.h"
#include "tc_issue.cuh"

namespace {
using namespace pxl;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kM = 128, kKeys = 2 * kM, kCols = 128;
constexpr int kGroups = 4, kProducerWarp = 4 * kGroups, kMmaWarp = kProducerWarp + 1, kThreads = (kMmaWarp + 1) * 32;
constexpr int kHalf = 128 * 128;
constexpr int kBufs = kGroups;  // of S: 2 t + (i & 1) has the scores of keys 128 t and on with unit i
constexpr int kUnits = 4;       // in the rings of queries and of their logarithms

template <int D>
struct Shape {
  static constexpr int kTile = D / 64 * kHalf;
  static constexpr int kOffQ = 2 * kTile;
  static constexpr int kOffLse = kOffQ + kUnits * kTile;   // [kUnits][128] floats
  static constexpr int kOffSums = kOffLse + kUnits * 512;  // [2][128] floats
  static constexpr int kOffBars = kOffSums + 2 * 512;
  static constexpr int kSmem = 1024 + kOffBars + 256;
  static constexpr uint32_t kIdesc = umma_idesc(kM, kCols, 1, 1);  // bf16
};
static_assert(Shape<128>::kSmem <= 232448);

struct Args {
  const int8_t* k_cache;
  const float2* kv_max;
  const int *block_tables, *cu_q, *ctx_lens, *seq_slots;
  const float* lse;  // log2 of the sums, [T, Hq]
  float *weights, *parts;
  int64_t W;
  int slots, T, max_q_len, Hq, Hkv, page, max_blocks, max_ctx, splits;
  int64_t num_blocks;
  float scale_log2;
  int window;
  int* status;
};

__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t four, int at, float unit) {
  return pack_bf16x2(static_cast<int8_t>(four >> (8 * at)) * unit, static_cast<int8_t>(four >> (8 * at + 8)) * unit);
}
// the power of two in what a code is multiplied by (within 2^100 of 1: 2^7 times it, and its inverse, are numbers), and the inverse of that
__device__ __forceinline__ float unit_of(float factor, float& inverse) {
  const uint32_t e = min(max(__float_as_uint(factor) >> 23 & 255u, 27u), 227u);
  inverse = __uint_as_float((254u - e) << 23);
  return __uint_as_float(e << 23);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_i8_weigh_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ Args a) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sm0 = smem_u32(smem);
  float* lse_sm = reinterpret_cast<float*>(smem + S::kOffLse);
  float* sum_sm = reinterpret_cast<float*>(smem + S::kOffSums);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
  // q_full, q_empty, lse_empty [kUnits] | s_full, s_empty [kBufs]
  const uint32_t q_full = smem_u32(bars), q_empty = q_full + 8 * kUnits, lse_empty = q_empty + 8 * kUnits, s_full = lse_empty + 8 * kUnits,
                 s_empty = s_full + 8 * kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kUnits + 2 * kBufs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  pdl_wait();

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y % a.Hkv, split = blockIdx.y / a.Hkv, G = a.Hq / a.Hkv;
  const int q_begin = a.cu_q[b], L = a.cu_q[b + 1] - q_begin, ctx = a.ctx_lens[b], slot = a.seq_slots ? a.seq_slots[b] : b;
  const int per_unit = kCols / G;
  const int key0 = blockIdx.x * kKeys, pos0 = ctx - L;  // position of the first query
  // uniform for the CTA, before any barrier or allocation; of a sequence that the attention reported there are no logarithms
  if (L <= 0 || key0 >= ctx || q_begin < 0 || q_begin > a.T - L || L > a.max_q_len) return;
  if (slot < 0 || slot >= a.slots || ctx > a.W || ctx > a.max_ctx) {
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, slot < 0 || slot >= a.slots ? PXL_DEV_BAD_SLOT : PXL_DEV_BAD_INDEX);
    return;
  }
  // units of queries that see some of the keys: positions key0 .. key0 + 255 + window - 1
  const int from = key0 - pos0 > 0 ? (key0 - pos0) / per_unit : 0;
  int past = L;  // first query behind every window
  if (a.window > 0 && static_cast<int64_t>(key0) + kKeys - 1 + a.window - pos0 < L) past = key0 + kKeys - 1 + a.window - pos0;
  const int all = past > 0 ? max(ceil_div(past, per_unit) - from, 0) : 0, each = ceil_div(all, a.splits);
  const int u_begin = from + min(split * each, all), n_units = __shfl_sync(0xffffffffu, min(each, from + all - u_begin), 0);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kUnits; ++s) {
      mbar_init(q_full + 8 * s, 1 + 32);  // the bytes, and the producer's lanes
      mbar_init(q_empty + 8 * s, 1);
      mbar_init(lse_empty + 8 * s, 8);    // the warps that take the unit
    }
    for (int s = 0; s < kBufs; ++s) {
      mbar_init(s_full + 8 * s, 1);
      mbar_init(s_empty + 8 * s, 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_q);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), kBufs * kCols);
    tmem_relinquish();
  }
  // the keys' codes as bf16, and zeros in the rows that no box of queries covers
  const int* bt = a.block_tables + static_cast<size_t>(b) * a.max_blocks;
  auto head_of = [&](int t) -> int64_t {  // page and head of token t, -1 off the cache or the context
    const int p = t / a.page, blk = t < ctx && p < a.max_blocks ? bt[p] : -1;
    if (blk >= 0 && blk < a.num_blocks) return static_cast<int64_t>(blk) * a.Hkv + kvh;
    if (t < ctx && a.status) atomicCAS(a.status, 0, PXL_DEV_BAD_BLOCK_PREFILL);
    return -1;
  };
  for (int i = threadIdx.x; i < kKeys * (D / 16); i += kThreads) {
    const int r = i / (D / 16), c = i % (D / 16);
    const int64_t head = head_of(key0 + r);
    uint4 x = make_uint4(0, 0, 0, 0);
    float unit = 0.f, inverse;
    if (head >= 0) {
      x = *reinterpret_cast<const uint4*>(a.k_cache + (head * a.page + (key0 + r) % a.page) * D + c * 16);
      unit = unit_of(a.kv_max[head].x * kInv127 * a.scale_log2, inverse);
    }
    const uint32_t w[4] = {x.x, x.y, x.z, x.w}, at = sm0 + (r / kM) * S::kTile + (c >> 2) * kHalf + r % kM * 128;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + ((((c & 3) * 2 + p) ^ (r & 7)) << 4)), "r"(codes_bf16x2(w[2 * p], 0, unit)),
                   "r"(codes_bf16x2(w[2 * p], 2, unit)), "r"(codes_bf16x2(w[2 * p + 1], 0, unit)), "r"(codes_bf16x2(w[2 * p + 1], 2, unit))
                   : "memory");
  }
  for (int i = threadIdx.x; i < kUnits * (D / 64) * (kCols - per_unit * G) * 8; i += kThreads) {
    const int c = i % 8, r = per_unit * G + i / 8 % (kCols - per_unit * G), h = i / 8 / (kCols - per_unit * G);
    st_shared_zero16(sm0 + S::kOffQ + h * kHalf + r * 128 + c * 16);
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_launch_dependents();
  const uint32_t tm_s = *tmem_slot;

  if (warp == kProducerWarp) {
    // logarithms of four units are on their way
    bool ok = true;
    float next[kUnits][4];
    auto load = [&](int i, float (&to)[4]) {  // of the unit's rows; none (infinity: a weight of 0) for rows that are nobody's
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j * 32 + lane, tok = (u_begin + i) * per_unit + r / G;
        to[j] = i < n_units && r < per_unit * G && tok < L ? a.lse[static_cast<int64_t>(q_begin + tok) * a.Hq + kvh * G + r % G] : INFINITY;
      }
    };
#pragma unroll
    for (int s = 0; s < kUnits; ++s) load(s, next[s]);
    for (int i0 = 0; ok && i0 < n_units; i0 += kUnits) {
#pragma unroll
      for (int s = 0; s < kUnits; ++s) {
        const int i = i0 + s;
        if (!ok || i >= n_units) break;
        if (i >= kUnits) ok = mbar_wait_bounded(q_empty + 8 * s, (i / kUnits - 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_EMPTY);
        if (ok && i >= kUnits) ok = mbar_wait_bounded(lse_empty + 8 * s, (i / kUnits - 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_EMPTY);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) lse_sm[s * 128 + j * 32 + lane] = -next[s][j];
        const uint32_t bar = q_full + 8 * s;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, (D / 64) * per_unit * G * 128);
          for (int h = 0; h < D / 64; ++h)
            tma_load_3d(sm0 + S::kOffQ + s * S::kTile + h * kHalf, &tm_q, bar, h * 64, kvh * G, q_begin + (u_begin + i) * per_unit);
        }
        mbar_arrive(bar);
        load(i + kUnits, next[s]);
      }
    }
  } else if (warp == kMmaWarp) {
    const uint32_t leader = elect_leader();
    bool ok = true;
    for (int i = 0; ok && i < n_units; ++i) {
      const int s = i % kUnits;
      ok = wait_warp(q_full + 8 * s, (i / kUnits) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_FULL);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int buf = 2 * t + (i & 1);
        if (ok && i >= 2) ok = wait_warp(s_empty + 8 * buf, ((i >> 1) - 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 32;
          mma_ss(tm_s + buf * kCols, umma_desc_k_sw128(sm0 + t * S::kTile + off), umma_desc_k_sw128(sm0 + S::kOffQ + s * S::kTile + off),
                 S::kIdesc, ks > 0 ? 1u : 0u, leader);
        }
        if (t == 1) commit(q_empty + 8 * s, leader);
        commit(s_full + 8 * buf, leader);
      }
    }
  }
  float total = 0.f;
  const int group = warp >> 2, r = (warp & 3) * 32 + lane, tile0 = key0 + (group >> 1) * kM, t = tile0 + r;  // this thread's key
  int failed = 0;
  if (warp < 4 * kGroups) {
    const int64_t head = head_of(t);
    float scale = head >= 0 ? a.kv_max[head].x * kInv127 * a.scale_log2 : 0.f, inverse;  // what the power of two leaves of it
    unit_of(scale, inverse);
    scale *= inverse;
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint64_t scale2 = pair2(scale, scale);
    for (int i = group & 1; i < n_units; i += 2) {
      const int buf = group, tok0 = (u_begin + i) * per_unit;
      failed = mbar_wait_bounded(s_full + 8 * buf, (i >> 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_TMEM_FULL) ? 0 : 1;
      failed = __any_sync(0xffffffffu, failed);  // warp-uniform: the TMEM loads below are warp-wide
      if (failed) break;
      tc_fence_after_sync();
      const int last = min(tok0 + per_unit, L) - 1;  // the unit's last query
      const bool interior = tile0 + kM - 1 <= pos0 + tok0 && (a.window <= 0 || tile0 > pos0 + last - a.window) && tok0 + per_unit <= L;
      // columns whose queries see this key
      const int first_tok = max(t - pos0 - tok0, 0), end_tok = min(last + 1 - tok0, a.window > 0 ? t - pos0 - tok0 + a.window : last + 1 - tok0);
      const int c_lo = min(first_tok, per_unit) * G, c_hi = head >= 0 ? max(end_tok, 0) * G : 0;
      const float4* neg = reinterpret_cast<const float4*>(lse_sm + i % kUnits * 128);
      uint64_t sum[2] = {0ull, 0ull};
      // 16 columns at a time, the next 16 scores and logarithms on their way
      uint32_t v[2][16];
      float4 z[2][4];
      auto load = [&](int c, uint32_t (&to)[16], float4 (&neg_lse)[4]) {
        tmem_ld_32x32b_x16(tm_s + buf * kCols + lane_sel + c, to);
#pragma unroll
        for (int j = 0; j < 4; ++j) neg_lse[j] = neg[(c >> 2) + j];
      };
      load(0, v[0], z[0]);
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        const int at = (c >> 4) & 1;
        tmem_ld_wait();
        if (c + 16 < kCols) load(c + 16, v[at ^ 1], z[at ^ 1]);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4& n = z[at][j >> 2];
          const float2 x = unpair2(fma2(pair2(__uint_as_float(v[at][j]), __uint_as_float(v[at][j + 1])), scale2, pair2(n.x, n.y)));
          const float2 y = unpair2(fma2(pair2(__uint_as_float(v[at][j + 2]), __uint_as_float(v[at][j + 3])), scale2, pair2(n.z, n.w)));
          float p[4] = {fast_exp2(x.x), fast_exp2(x.y), fast_exp2(y.x), fast_exp2(y.y)};
          if (!interior) {
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = c + j + k >= c_lo && c + j + k < c_hi ? p[k] : 0.f;
          }
          sum[0] = add2(sum[0], pair2(p[0], p[1]));
          sum[1] = add2(sum[1], pair2(p[2], p[3]));
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(s_empty + 8 * buf);
        mbar_arrive(lse_empty + 8 * (i % kUnits));
      }
      const float2 two = unpair2(add2(sum[0], sum[1]));
      total += two.x + two.y;
    }
    if (group & 1) sum_sm[(group >> 1) * 128 + r] = total;
  }

  __syncwarp();
  if (*abort_flag) __nanosleep(200000);  // loads that are still in flight must land before smem is released
  tc_fence_before_sync();
  if (!__syncthreads_or(failed) && warp < 4 * kGroups && !(group & 1) && t < ctx) {
    total += sum_sm[(group >> 1) * 128 + r];
    if (a.splits == 1) atomicAdd(a.weights + (static_cast<int64_t>(slot) * a.Hkv + kvh) * a.W + t, total);  // (another may have the slot)
    else a.parts[((static_cast<int64_t>(split) * gridDim.z + b) * a.Hkv + kvh) * a.max_ctx + t] = total;
  }
  tc_fence_after_sync();
  if (warp == kMmaWarp) tmem_dealloc(tm_s, kBufs * kCols);
}

// Adds up the parts of split sums.
__global__ void __launch_bounds__(256) attn_i8_weigh_join_kernel(const __grid_constant__ Args a) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x, ctx = a.ctx_lens[b], slot = a.seq_slots ? a.seq_slots[b] : b;
  const int q_begin = a.cu_q[b], L = a.cu_q[b + 1] - q_begin;
  if (t >= ctx || L <= 0 || q_begin < 0 || q_begin > a.T - L || L > a.max_q_len || slot < 0 || slot >= a.slots || ctx > a.W || ctx > a.max_ctx) return;
  float sum = 0.f;
  for (int s = 0; s < a.splits; ++s) sum += a.parts[((static_cast<int64_t>(s) * gridDim.z + b) * a.Hkv + h) * a.max_ctx + t];
  atomicAdd(a.weights + (static_cast<int64_t>(slot) * a.Hkv + h) * a.W + t, sum);
}

// CTAs that share the queries of a tile of keys: enough to fill the chip, each with at least eight units.
int splits_of(int B, int max_q_len, int Hq, int Hkv, int max_ctx) {
  const int64_t tiles = static_cast<int64_t>(ceil_div(max_ctx, kKeys)) * Hkv * B;
  const int64_t fill = pxl_host::num_sms() / (tiles > 0 ? tiles : 1), most = max_q_len / (kCols / (Hq / Hkv)) / 8;
  const int64_t s = fill < most ? fill : most;
  return s < 1 ? 1 : static_cast<int>(s);
}

template <int D>
int launch_weigh(const CUtensorMap& tq, const Args& a, int B, cudaStream_t stream) {
  static std::atomic<bool> configured[64];  // function attributes are per device
  std::atomic<bool>& done = configured[pxl_host::current_device_slot()];
  if (!done.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(attn_i8_weigh_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem) != cudaSuccess)
      return PXL_ERR_CUDA;
    done.store(true, std::memory_order_relaxed);
  }
  pxl_host::launch(attn_i8_weigh_kernel<D>, dim3(ceil_div(a.max_ctx, kKeys), a.Hkv * a.splits, B), dim3(kThreads), Shape<D>::kSmem, stream, tq, a);
  if (a.splits > 1)
    pxl_host::launch_behind(attn_i8_weigh_join_kernel, dim3(ceil_div(a.max_ctx, 256), a.Hkv, B), dim3(256), 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

}  // namespace

PXL_EXPORT int64_t pxl_attn_i8_weigh_workspace(int B, int max_q_len, int Hq, int Hkv, int max_ctx) {
  if (B <= 0 || Hkv <= 0 || Hq < Hkv || max_q_len < 0 || max_ctx <= 0) return 0;
  const int s = splits_of(B, max_q_len, Hq, Hkv, max_ctx);
  return s > 1 ? static_cast<int64_t>(s) * B * Hkv * max_ctx * 4 : 0;
}

PXL_EXPORT int pxl_attn_i8_weigh(const void* q, int64_t q_stride, const void* k_cache, const float* kv_max, const int* block_tables,
                                 const int* cu_q, const int* ctx_lens, const float* lse, float* weights, int64_t W, int slots,
                                 const int* seq_slots, void* workspace, int64_t workspace_bytes, int T, int B, int max_q_len, int Hq, int Hkv,
                                 int D, int page, int max_blocks, int64_t num_blocks, float scale, int window, int max_ctx, int* status,
                                 cudaStream_t stream) {
  if (T <= 0 || B <= 0) return PXL_OK;
  if ((D != 64 && D != 128) || (page != 16 && page != 32 && page != 64) || Hkv <= 0 || Hq % Hkv || Hq / Hkv < 1 || Hq / Hkv > 16 ||
      !(scale > 0.f) || (q_stride & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache)) & 15) ||
      (reinterpret_cast<uintptr_t>(kv_max) & 7) || max_blocks <= 0 || max_q_len < 0 || max_ctx <= 0 || max_ctx >= (1 << 30) ||
      window < 0 || window > (1 << 30) || num_blocks <= 0 ||
      !lse || !weights)
    return PXL_ERR_INVALID_ARG;
  const int splits = splits_of(B, max_q_len, Hq, Hkv, max_ctx);
  const int64_t need = pxl_attn_i8_weigh_workspace(B, max_q_len, Hq, Hkv, max_ctx);
  if (workspace_bytes < need || (need > 0 && !workspace)) return PXL_ERR_INVALID_ARG;
  if (static_cast<int64_t>(Hkv) * splits > 65535 || B > 65535) return PXL_ERR_TOO_LARGE;
  CUtensorMap tq;
  if (!pxl_host::make_tmap_queries(&tq, q, q_stride, T, Hq, D, Hq / Hkv)) return PXL_ERR_TENSORMAP;
  const Args a{static_cast<const int8_t*>(k_cache), reinterpret_cast<const float2*>(kv_max), block_tables, cu_q, ctx_lens, seq_slots, lse,
               weights, static_cast<float*>(workspace), W, slots, T, max_q_len, Hq, Hkv, page, max_blocks, max_ctx, splits, num_blocks, scale * kLog2e,
               window, status};
  return D == 64 ? launch_weigh<64>(tq, a, B, stream) : launch_weigh<128>(tq, a, B, stream);
}
