// Decode attention over keys and values in 8 bits (layout: kv_i8.cu): one query per sequence.
//
// Every CTA gets the same number of tiles of 64 keys of the row of all (sequence, key head) pairs (attention_walk.cuh). A producer warp
// brings the codes by TMA, page by page, and the pages' magnitudes by 8-byte cp.async into the same stage; four consumer warps, two per
// tile, convert the codes where they multiply them (mma.sync, f16). Keys, and columns of the values, are the 16 rows of the products, the
// query heads of a key head their 8 columns (twice where there are more): S^T = K q^T, O^T = V^T P^T, a transposition of 8 x 8 between them.
// A score is multiplied by its page's key magnitude with the softmax scale. Values are held relative to R, at least the largest value
// magnitude so far and at most twice as much when it was chosen: an exponential is taken of the score plus log2 of the page's share of R,
// so that what is rounded to f16 (2^-11) is the probability times the share; a factor of 2^11 keeps its bits down to 2^-25 of the row's
// largest, and it is rounded in steps of 2^-35 below. The reference maximum may lag by 2^4 before anything is rescaled.
// What bounds it is memory: 128 sequences of up to 12000 tokens, 40 heads on 8, 305 us with the join, 6.5 TB/s (calls one behind the other 308
// to 361 on four cards). Two to four CTAs per SM, since a tile's products wait for its exponentials; f16 rather than 8-bit products, since q
// and the probabilities would lose bits. Short pairs are bound by their beginning and end (203 windows of 128 keys, 64 heads of 64: 22 us).
// A pair that lies in several CTAs is added up by a second kernel; short ones are not cut, and few pairs get a cluster each, whose CTAs add
// up from each other's shared memory (one sequence of up to 776 tokens, 32 heads of 128: 9.9 -> 6.7 us). Where the weights are wanted, the
// scores go to the workspace (4 bytes per query head and key beside 2 D per key head) and a third kernel adds their exponentials once the sums are
// known.
#include <atomic>
#include <type_traits>

#include "attention_walk.cuh"
#include "common.cuh"
#include "kv_i8.cuh"
#include "pxl_api.h"
#include "tc_issue.cuh"

namespace {
using namespace pxl;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 160;  // four consumer warps and the producer

constexpr float kUp = 11.f;    // log2 of the factor on probabilities in f16
constexpr float kLag = 4.f;    // log2 of how far the reference maximum may lag

// (Heads of 64, 40 sequences of up to 8000 tokens, 32 heads: three CTAs of eight stages 62 us, four of six 59.)
constexpr int ctas_per_sm(int D, int NH) { return NH > 1 ? 2 : D == 64 ? 4 : 3; }

// NH: tiles of 8 query heads
template <int D, int NH>
struct Shape {
  static constexpr int kCtas = ctas_per_sm(D, NH);
  static constexpr int kTileBytes = kKeyTile * D;                // of K, or of V
  static constexpr int kStages = D == 128 ? 4 : NH == 1 ? 6 : 8;  // even: a stage belongs to one pair of warps
  static constexpr int kVecs = NH * D / 16;                      // 16-byte vectors of a lane's output
  static constexpr int kStats = 16 * NH + 4;                     // maxima and sums of a warp's heads, R
  static constexpr int kOffParts = kStages * 2 * kTileBytes;     // [4][kVecs / 2][32] float4
  static constexpr int kOffStats = kOffParts + 2 * kVecs * 512;  // [4][kStats] floats
  static constexpr int kOffMax = kOffStats + 4 * kStats * 4;     // [stages][4] magnitudes of a stage's pages
  static constexpr int kOffBars = kOffMax + kStages * 32;
  static constexpr int kSmem = 1024 + kOffBars + kStages * 16 + 16;
  static_assert(kCtas * (kSmem + 1024) <= 233472);
};

struct Args {
  const bf16* q;
  int64_t q_stride;
  const float2* kv_max;
  const int *block_tables, *ctx_lens;
  bf16* out;
  int64_t out_stride;
  const float* sinks;
  float *parts, *lse, *scores;  // workspace: partial results, log2 of the sums [B, Hq], scores [B, Hq, score_stride]
  int64_t score_stride;
  int B, Hq, Hkv, page, max_blocks;
  int64_t num_blocks;
  float scale_log2;
  int window;
  bool uncut;
  int log_ranks;  // of the CTAs of a cluster that has a pair to itself; 0: none
  int* status;
};

__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// arrives once the copies that this thread began are there; the barrier counts the arrival
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// largest of, and sum over, the lanes that have the same heads
__device__ __forceinline__ float keys_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float keys_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Lane 4 g + t has keys g and g + 8 of a product, heads 2 t and 2 t + 1 of a tile of heads, columns 16 c + 2 g and + 1 of the output.
template <int D, int NH>
struct Rows {
  static constexpr int kKeys = 32, kSteps = D / 16;
  uint32_t qf[NH][kSteps][2];
  float row_scale[NH][2], o[NH][D / 16][4], m_run[NH][2], l_run[NH][2], r_run, log_r;
  bool none;  // values without a magnitude were seen

  // byte offset of 16-byte chunk c of a row of a tile as TMA lays it down
  static __device__ __forceinline__ uint32_t chunk(int row, int c) {
    return D == 128 ? row * 128 + ((c ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  }

  // q: first query head of the key head. Lane t of a quad takes columns D / 4 * t and on, of q as of the keys.
  __device__ __forceinline__ void begin(const bf16* q, int G, float scale_log2) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int r = g8 + n * 8;
      uint2 x[kSteps];
      float mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        x[ks] = r < G ? *reinterpret_cast<const uint2*>(q + r * D + t4 * (D / 4) + ks * 4) : make_uint2(0, 0);
        const float2 a = unpack_bf16x2(x[ks].x), b = unpack_bf16x2(x[ks].y);
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(a.x)), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y)));
      }
      float down;
      const float up = row_up(quad_max(mx), down);
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        const float2 a = unpack_bf16x2(x[ks].x), b = unpack_bf16x2(x[ks].y);
        qf[n][ks][0] = pack_f16x2(a.x * up, a.y * up);
        qf[n][ks][1] = pack_f16x2(b.x * up, b.y * up);
      }
      down *= scale_log2 * kInv127;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[n][e] = __shfl_sync(0xffffffffu, down, (2 * t4 + e) * 4);
        m_run[n][e] = -INFINITY;
        l_run[n][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    r_run = 0.f;
    log_r = -INFINITY;
    none = false;
  }

  // Keys r0 .. r0 + 31 of a tile; the first is token tok_base. near, far: magnitudes of the pages of its first and second 16. scores: where
  // they go for row 0 of the pair (null: nowhere), a row `score_stride` behind the one before.
  __device__ __forceinline__ void step(uint32_t k_smem, uint32_t v_smem, int r0, int tok_base, int lo, int hi, float2 near, float2 far,
                                       float* scores, int64_t score_stride, int G) {
    if (!(tok_base < hi && tok_base + kKeys > lo)) return;  // warp-uniform
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    float s[NH][2][4];  // 16 keys each
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) s[n][k][0] = s[n][k][1] = s[n][k][2] = s[n][k][3] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint32_t w[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[j][0]), "=r"(w[j][1]), "=r"(w[j][2]), "=r"(w[j][3])
                     : "r"(k_smem + chunk(r0 + j * 8 + g8, t4 * (D / 64) + c)));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t x = flip_codes(w[2 * k][i]), y = flip_codes(w[2 * k + 1][i]);
          const uint32_t a[4] = {codes_f16x2<0x4140>(x), codes_f16x2<0x4140>(y), codes_f16x2<0x4342>(x), codes_f16x2<0x4342>(y)};
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_m16n8k16_f16(s[n][k], a, qf[n][c * 4 + i][0], qf[n][c * 4 + i][1]);
        }
    }
    const bool whole = tok_base + kKeys <= hi && tok_base >= lo;  // every token is seen
    bool out[2][2] = {{false, false}, {false, false}};            // of this lane's keys: not seen
    if (!whole) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int tok = tok_base + k * 16 + r * 8 + g8;
          out[k][r] = !(tok < hi && tok >= lo);
#pragma unroll
          for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[n][k][2 * r + e] = out[k][r] ? -INFINITY : s[n][k][2 * r + e];
        }
    }
    // R, of pages that have a token which is seen (a NaN is passed over: it is for the output, not for the sum); the maxima
    const float near_y = tok_base + 16 > lo ? near.y : 0.f, far_y = tok_base + 16 < hi ? far.y : 0.f, most = fmaxf(near_y, far_y);
    none = none || near_y + far_y != near_y + far_y;
    float mx[NH][2];
    bool grow = most > r_run;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[n][e] = fmaxf(fmaxf(s[n][0][e], s[n][0][2 + e]) * (row_scale[n][e] * near.x), fmaxf(s[n][1][e], s[n][1][2 + e]) * (row_scale[n][e] * far.x));
        grow = grow || mx[n][e] > m_run[n][e] + kLag;
      }
    if (__any_sync(0xffffffffu, grow)) {
      float r_corr = 1.f;
      if (most > r_run) {
        const float r_new = fminf(2.f * most, 3.3e38f);
        r_corr = page_share(r_run, r_new);
        r_run = r_new;
        log_r = __log2f(r_new);
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m_new = fmaxf(m_run[n][e], keys_max(mx[n][e]));
          const float corr = fast_exp2(m_run[n][e] - ((m_new == -INFINITY) ? 0.f : m_new));
          m_run[n][e] = m_new;
          l_run[n][e] *= corr;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[n][i][e] *= corr * r_corr, o[n][i][2 + e] *= corr * r_corr;
        }
    }
    const float up[2] = {kUp + page_log(near.y, log_r), kUp + page_log(far.y, log_r)};
    const float down[2] = {fast_exp2(-up[0]), fast_exp2(-up[1])};
    uint32_t pf[NH][2][2];  // [16 keys][8 of them], transposed: heads are rows
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const float m_use[2] = {m_run[n][0] == -INFINITY ? 0.f : m_run[n][0], m_run[n][1] == -INFINITY ? 0.f : m_run[n][1]};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float page = k == 0 ? near.x : far.x;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float scale = row_scale[n][e] * page, off = up[k] - m_use[e];
          const int head = n * 8 + 2 * t4 + e;
          if (scores && head < G) {
            float* to = scores + head * score_stride + tok_base + k * 16 + g8;
            to[0] = s[n][k][e] * scale;
            to[8] = s[n][k][2 + e] * scale;
          }
          float p0 = fast_exp2(fmaf(s[n][k][e], scale, off)), p1 = fast_exp2(fmaf(s[n][k][2 + e], scale, off));
          if (!whole) {  // (a magnitude that is zero, or none, of a token that is not seen)
            p0 = out[k][0] ? 0.f : p0;
            p1 = out[k][1] ? 0.f : p1;
          }
          const float both = p0 + p1;
          l_run[n][e] += both == 0.f ? 0.f : both * down[k];
          s[n][k][e] = p0;
          s[n][k][2 + e] = p1;
        }
        pf[n][k][0] = transpose_8x8(pack_f16x2(s[n][k][0], s[n][k][1]));
        pf[n][k][1] = transpose_8x8(pack_f16x2(s[n][k][2], s[n][k][3]));
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int mi = lane >> 3, row = r0 + k * 16 + (mi & 1) * 8 + (lane & 7);
#pragma unroll
      for (int c = 0; c < D / 16; c += 2) {  // 16 columns per chunk; a transposed pair of bytes is two columns of a token
        uint32_t r[4];                       // chunk c: tokens 0-7, 8-15; chunk c + 1: the same
        ldmatrix_x4_trans(r, v_smem + chunk(row, c + (mi >> 1)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = flip_codes(r[2 * h]), y = flip_codes(r[2 * h + 1]);
          const uint32_t a[4] = {codes_f16x2<0x4240>(x), codes_f16x2<0x4341>(x), codes_f16x2<0x4240>(y), codes_f16x2<0x4341>(y)};
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_m16n8k16_f16(o[n][c + h], a, pf[n][k][0], pf[n][k][1]);
        }
      }
    }
  }
};

// What two parts of a pair's keys have of a row: o in units of R, relative to the maximum.
struct Joined {
  float fa, fb;  // factors on the outputs
  __device__ __forceinline__ Joined(float& m, float& l, float r, float r_new, float m2, float l2, float r2) {
    const float M = fmaxf(m, m2), Mu = M == -INFINITY ? 0.f : M;
    fa = fast_exp2(m - Mu);
    fb = fast_exp2(m2 - Mu);
    l = l * fa + l2 * fb;
    m = M;
    fa *= page_share(r, r_new);
    fb *= page_share(r2, r_new);
  }
};
// R / sum, and log2 of the sum of exponentials, for a row with a sink or without
__device__ __forceinline__ float finish(float M, float L, float R, float sink, float& lse) {
  const float Mx = fmaxf(M, sink), Mu = Mx == -INFINITY ? 0.f : Mx;
  const float e = fast_exp2(M - Mu), denom = L * e + fast_exp2(sink - Mu);
  lse = denom == 0.f ? INFINITY : Mu + __log2f(denom);
  return denom == 0.f ? 0.f : __fdividef(e, denom) * (R * (kInv127 * 0x1p-11f));
}

// TOGETHER: a cluster of 2^a.log_ranks CTAs has a pair, and adds its parts up from shared memory.
constexpr int kLogRanks = 3, kRanks = 1 << kLogRanks;  // at most
template <int D, int NH, bool TOGETHER>
__global__ void __launch_bounds__(kThreads, Shape<D, NH>::kCtas)
attn_i8_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using S = Shape<D, NH>;
  using R = Rows<D, NH>;
  constexpr int STAGES = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t stage0 = smem_u32(smem);  // stage s: K at s * 2 * kTileBytes, V behind it
  float4* parts = reinterpret_cast<float4*>(smem + S::kOffParts);
  float* stats = reinterpret_cast<float*>(smem + S::kOffStats);
  const float2* max_sm = reinterpret_cast<const float2*>(smem + S::kOffMax);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);  // full[S], empty[S]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * STAGES);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const int G = a.Hq / a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int shift = a.page == 16 ? 2 : a.page == 32 ? 1 : 0, ppt = 1 << shift;  // pages per tile

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1 + ppt);  // the bytes, and the magnitudes of each page
      mbar_init(empty0 + 8 * s, 2);       // one arrival per warp that reads the stage
    }
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // the lengths and the tables of a step are there before its first kernel, the queries and the new keys after the wait
  const DecodeWork work{a.ctx_lens, a.B, a.Hkv, a.window, 0};
  const int rank = static_cast<int>(blockIdx.x) & ((1 << a.log_ranks) - 1);
  DecodeWalk walk = [&] {
    if constexpr (TOGETHER) return DecodeWalk(work, PairShare{static_cast<int>(blockIdx.x) >> a.log_ranks, rank, a.log_ranks});
    else return DecodeWalk(work, blockIdx.x, gridDim.x, a.uncut);
  }();
  const int pair_b = walk.b, pair_kvh = walk.kvh;
  const bool idle = walk.left <= 0;
  auto blocks_of = [&](const DecodeWalk& w) {
    return TileBlocks{a.block_tables + static_cast<size_t>(w.left > 0 ? w.b : 0) * a.max_blocks, w.tiles, w.t, w.left > 0 ? w.count() : 0,
                      a.page, shift, w.hi, a.max_blocks, a.num_blocks, a.status};
  };
  TileBlocks blocks = blocks_of(walk);
  if (warp == 4) blocks.begin();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  int failed = 0;
  int g = 0;  // tiles so far: tile g is in stage g % STAGES
  if (warp == 4) {  // producer: lane p issues the boxes of page p of the tile
    while (walk.left > 0 && !failed) {
      const int n = walk.count(), kvh = walk.kvh;
      walk.next();
      TileBlocks ahead = blocks_of(walk);
      ahead.begin();  // in flight during this pair
      for (int it = 0; it < n; ++it, ++g) {
        const int stage = g % STAGES;
        const int blk = blocks(it);
        int okf = 1;
        if (g >= STAGES && lane == 0)
          okf = mbar_wait_bounded(empty0 + 8 * stage, ((g / STAGES) - 1) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_EMPTY) ? 1 : 0;
        okf = __shfl_sync(0xffffffffu, okf, 0);
        if (!okf) {
          failed = 1;
          break;
        }
        const uint32_t bar = full0 + 8 * stage;
        const uint32_t dst = stage0 + stage * 2 * S::kTileBytes + lane * a.page * D;
        if (lane == 0) mbar_arrive_expect_tx(bar, 2 * S::kTileBytes);
        __syncwarp();
        if (lane < ppt) {
          const int head = blk * a.Hkv + kvh;
          tma_load_2d(dst, &tm_k, bar, 0, head * a.page);
          tma_load_2d(dst + S::kTileBytes, &tm_v, bar, 0, head * a.page);
          cp_async_8(stage0 + S::kOffMax + stage * 32 + lane * 8, a.kv_max + head);
          cp_async_arrive(bar);
        }
      }
      blocks = ahead;
    }
  } else {
    R rows;
    const int r0 = (warp & 1) * R::kKeys;
    // pages of the first and second 16 of the warp's keys among those of the tile
    const int near = r0 >> (6 - shift), far = (r0 + 16) >> (6 - shift);
    // after a failed wait the warp goes on to the end without loads or products: the others meet it at the barriers
    for (; walk.left > 0; walk.next()) {
      const int n = walk.count(), head0 = walk.kvh * G;
      rows.begin(a.q + walk.b * a.q_stride + head0 * D, G, a.scale_log2);
      float* scores = a.scores ? a.scores + (static_cast<int64_t>(walk.b) * a.Hq + head0) * a.score_stride : nullptr;
      if (lane < 2 * G && walk.left > walk.take) {  // the next pair's queries, to be near when they are wanted
        const int kvh = walk.kvh + 1 < a.Hkv ? walk.kvh + 1 : 0, b = walk.b + (kvh == 0 ? 1 : 0);
        if (lane * 64 < G * D) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.q + b * a.q_stride + kvh * G * D + lane * 64));
      }
      for (int it = 0; it < n; ++it, ++g) {
        if ((g & 1) != (warp >> 1)) continue;  // warps 0 and 1 take the even stages, 2 and 3 the odd ones
        const int stage = g % STAGES;
        if (!failed)
          failed = __any_sync(0xffffffffu, !mbar_wait_bounded(full0 + 8 * stage, (g / STAGES) & 1, abort_flag, a.status, PXL_DEV_TIMEOUT_FULL));
        if (failed) continue;
        const uint32_t k_smem = stage0 + stage * 2 * S::kTileBytes;
        const int tok = walk.tiles[walk.t + it] * kKeyTile + r0;
        rows.step(k_smem, k_smem + S::kTileBytes, r0, tok, walk.lo, walk.hi, max_sm[stage * 4 + near], max_sm[stage * 4 + far],
                  tok + R::kKeys <= a.score_stride ? scores : nullptr, a.score_stride, G);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * stage);
      }

      if (rows.none) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) rows.o[n][i][0] = rows.o[n][i][1] = rows.o[n][i][2] = rows.o[n][i][3] = NAN;
      }
      // The four warps' results, each of some keys, become a quarter of the columns of all keys each: half of them change hands with the warp
      // that had the other tiles, half of the rest with the one that had the other 32 keys of these. A warp writes its second gift where it
      // has read the first one.
      float sums[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) sums[n][0] = keys_sum(rows.l_run[n][0]), sums[n][1] = keys_sum(rows.l_run[n][1]);
      const int t4 = lane & 3;
      auto exchange = [&](auto half, int at, int from, bool upper) {  // keeps `half` of 2 * half vectors
        constexpr int N = decltype(half)::value;
        float4* to = parts + at * (S::kVecs / 2) * 32 + lane;
        float* st = stats + at * S::kStats;
#pragma unroll
        for (int n = 0; n < NH; ++n) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float (&lo)[4] = rows.o[n][i], (&hi)[4] = rows.o[n][i + N];
            to[(n * N + i) * 32] = upper ? make_float4(lo[0], lo[1], lo[2], lo[3]) : make_float4(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = upper ? hi[j] : lo[j];
          }
          if (lane < 4)
            *reinterpret_cast<float4*>(st + n * 16 + lane * 4) = make_float4(rows.m_run[n][0], sums[n][0], rows.m_run[n][1], sums[n][1]);
        }
        if (lane == 0) st[16 * NH] = rows.r_run;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const float4* of = parts + from * (S::kVecs / 2) * 32 + lane;
        const float* os = stats + from * S::kStats;
        const float r2 = os[16 * NH], r_new = fmaxf(rows.r_run, r2);
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const float4 other = *reinterpret_cast<const float4*>(os + n * 16 + t4 * 4);
          const Joined x(rows.m_run[n][0], sums[n][0], rows.r_run, r_new, other.x, other.y, r2);
          const Joined y(rows.m_run[n][1], sums[n][1], rows.r_run, r_new, other.z, other.w, r2);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float4 v = of[(n * N + i) * 32];
            float (&o)[4] = rows.o[n][i];
            o[0] = o[0] * x.fa + v.x * x.fb;
            o[1] = o[1] * y.fa + v.y * y.fb;
            o[2] = o[2] * x.fa + v.z * x.fb;
            o[3] = o[3] * y.fa + v.w * y.fb;
          }
        }
        rows.r_run = r_new;
        __syncwarp();  // all lanes have read the sums
      };
      exchange(std::integral_constant<int, D / 32>(), warp, warp ^ 2, (warp & 2) != 0);
      exchange(std::integral_constant<int, D / 64>(), warp ^ 2, warp ^ 3, (warp & 1) != 0);
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the places are free for the next pair
      const int g8 = lane >> 2, col = ((warp >> 1) * 2 + (warp & 1)) * (D / 4) + 2 * g8;
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = n * 8 + 2 * t4 + e;
          const float M = rows.m_run[n][e], L = sums[n][e];
          if (r >= G || failed) continue;
          if constexpr (TOGETHER) {
            float* po = reinterpret_cast<float*>(parts) + r * D + col;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) *reinterpret_cast<float2*>(po + i * 16) = make_float2(rows.o[n][i][e], rows.o[n][i][2 + e]);
            if (warp == 0 && g8 == 0) reinterpret_cast<float4*>(stats)[r] = make_float4(M, L, rows.r_run, 1.f);
          } else if (walk.whole()) {
            float lse;
            const float f = finish(M, L, rows.r_run, a.sinks ? a.sinks[head0 + r] * kLog2e : -INFINITY, lse);
            if (a.lse && warp == 0 && g8 == 0) a.lse[static_cast<size_t>(walk.b) * a.Hq + head0 + r] = lse;
            bf16* dst = a.out + walk.b * a.out_stride + (head0 + r) * D + col;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) *reinterpret_cast<uint32_t*>(dst + i * 16) = pack_bf16x2(rows.o[n][i][e] * f, rows.o[n][i][2 + e] * f);
          } else {
            float* po = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (walk.t == 0 ? 1 : 0)) * (G * (D + 2) + 4);
#pragma unroll
            for (int i = 0; i < D / 64; ++i)
              *reinterpret_cast<float2*>(po + r * D + i * 16 + col) = make_float2(rows.o[n][i][e], rows.o[n][i][2 + e]);
            if (warp == 0 && g8 == 0) po[G * D + r] = M, po[G * D + G + r] = L, po[G * (D + 2)] = rows.r_run;
          }
        }
    }
  }
  if constexpr (TOGETHER) {
    static_assert(4 * S::kStats >= 64 && S::kStats % 4 == 0 && 2 * S::kVecs * 128 >= 8 * NH * D);
    if (idle && threadIdx.x < G) reinterpret_cast<float4*>(stats)[threadIdx.x] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    __syncwarp();
    cluster_sync_all();
    // a rank's share of the results, four columns per thread
    const int ranks = 1 << a.log_ranks, all = G * D / 4, each = (all + ranks - 1) >> a.log_ranks;
    for (int i = threadIdx.x; i < each && rank * each + i < all; i += kThreads) {
      const int at = rank * each + i;
      const int r = at / (D / 4);
      float4 st[kRanks], o[kRanks];
      float M = -INFINITY, L = 0.f, top = 0.f;
#pragma unroll
      for (int k = 0; k < kRanks; ++k) {
        const uint32_t from = k < ranks ? k : 0;
        st[k] = ld_shared_cluster_f32x4(cluster_map_shared(smem_u32(stats) + r * 16, from));
        o[k] = ld_shared_cluster_f32x4(cluster_map_shared(smem_u32(parts) + at * 16, from));
        if (k >= ranks) st[k] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < kRanks; ++k) M = fmaxf(M, st[k].x), top = fmaxf(top, st[k].z);
      const float Mu = M == -INFINITY ? 0.f : M;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kRanks; ++k) {
        const float e = fast_exp2(st[k].x - Mu), f = e * page_share(st[k].z, top);
        L += st[k].y * e;
        if (st[k].w != 0.f) acc.x += o[k].x * f, acc.y += o[k].y * f, acc.z += o[k].z * f, acc.w += o[k].w * f;
      }
      const int head = pair_kvh * G + r;
      float lse;
      const float f = finish(M, L, top, a.sinks ? a.sinks[head] * kLog2e : -INFINITY, lse);
      if (a.lse && at % (D / 4) == 0) a.lse[static_cast<size_t>(pair_b) * a.Hq + head] = lse;
      *reinterpret_cast<uint2*>(a.out + pair_b * a.out_stride + head * D + at % (D / 4) * 4) =
          make_uint2(pack_bf16x2(acc.x * f, acc.y * f), pack_bf16x2(acc.z * f, acc.w * f));
    }
    __syncwarp();
    cluster_sync_all();  // nobody's shared memory goes before it has been read
  }
  if (__syncthreads_or(failed)) __nanosleep(200000);  // loads that are still in flight must land before the shared memory is released
}

// Adds up the pairs that lie in several CTAs. Block x: the pair that the border between CTAs x and x + 1 cuts, if no border before it does.
// First a warp per query head finds the factors of all parts, then every warp adds columns of a head at a time.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
attn_i8_join_kernel(const __grid_constant__ Args a, int ctas) {
  extern __shared__ float factor[];  // [G][parts]
  __shared__ float final_sm[16];
  const DecodeWork work{a.ctx_lens, a.B, a.Hkv, a.window, 0};
  const int cut = blockIdx.x + 1, G = a.Hq / a.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const DecodeShares at(work.total(), ctas);
  const int64_t pos = at[cut];
  int b, kvh, t;
  work.find(pos, b, kvh, t);
  const int64_t begin = pos - t;
  const bool mine = t > 0 && b < a.B && at[cut - 1] <= begin;
  int last = cut;  // CTA that ends the pair; all of them up to it have tiles of it
  if (mine)
    for (const int64_t end = begin + work.weight(b); at[last + 1] < end;) ++last;
  pdl_wait();
  pdl_launch_dependents();
  if (!mine) return;
  const int place = G * (D + 2) + 4, n = last - cut + 2;
  const float* first = a.parts + (static_cast<int64_t>(cut) * 2 - 1) * place;  // the end of CTA cut - 1; then the starts of the others
  auto part = [&](int x) { return first + (x == 0 ? 0 : (2 * x - 1) * static_cast<int64_t>(place)); };
  for (int g = warp; g < G; g += kJoinThreads / 32) {
    float M = -INFINITY, R = 0.f, L = 0.f;
    for (int x = lane; x < n; x += 32) M = fmaxf(M, part(x)[G * D + g]), R = fmaxf(R, part(x)[G * (D + 2)]);
    M = warp_reduce_max(M);
    R = warp_reduce_max(R);
    const float Mu = M == -INFINITY ? 0.f : M;
    for (int x = lane; x < n; x += 32) {
      const float f = fast_exp2(part(x)[G * D + g] - Mu);
      L += part(x)[G * D + G + g] * f;
      factor[g * n + x] = f * page_share(part(x)[G * (D + 2)], R);
    }
    L = warp_reduce_sum(L);
    const int head = kvh * G + g;
    float lse;
    const float f = finish(M, L, R, a.sinks ? a.sinks[head] * kLog2e : -INFINITY, lse);
    if (lane == 0) {
      final_sm[g] = f;
      if (a.lse) a.lse[static_cast<size_t>(b) * a.Hq + head] = lse;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D / 2; i += kJoinThreads) {
    const int g = i / (D / 2);
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int x = 0; x < n; ++x) {
      const float f = factor[g * n + x];
      const float2 v = *reinterpret_cast<const float2*>(part(x) + i * 2);
      acc.x += v.x * f, acc.y += v.y * f;
    }
    const float f = final_sm[g];
    *reinterpret_cast<uint32_t*>(a.out + b * a.out_stride + kvh * G * D + i * 2) = pack_bf16x2(acc.x * f, acc.y * f);
  }
}

// What every token got, from the scores and the sums.
constexpr int kWeighKeys = 1024;
__global__ void __launch_bounds__(256)
attn_i8_weigh_kernel(const __grid_constant__ Args a, float* __restrict__ weights, int64_t W, int slots, const int* __restrict__ seq_slots) {
  __shared__ float lse_sm[16];
  const int b = blockIdx.z, h = blockIdx.y, G = a.Hq / a.Hkv;
  const int ctx = a.ctx_lens[b], slot = seq_slots ? seq_slots[b] : b;
  const int lo = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
  const int t0 = blockIdx.x * kWeighKeys + threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x == 0 && threadIdx.x == 0 && h == 0 && ctx > 0 && a.status) {
    if (slot < 0 || slot >= slots) atomicCAS(a.status, 0, PXL_DEV_BAD_SLOT);
    else if (ctx > W || ctx > a.score_stride) atomicCAS(a.status, 0, PXL_DEV_BAD_INDEX);
  }
  if (slot < 0 || slot >= slots || ctx > W || ctx > a.score_stride || static_cast<int>(blockIdx.x) * kWeighKeys >= ctx ||
      static_cast<int>(blockIdx.x + 1) * kWeighKeys <= lo)
    return;
  if (threadIdx.x < G) lse_sm[threadIdx.x] = a.lse[static_cast<size_t>(b) * a.Hq + h * G + threadIdx.x];
  __syncthreads();
  float* w = weights + (static_cast<int64_t>(slot) * a.Hkv + h) * W;
  const float* s = a.scores + (static_cast<int64_t>(b) * a.Hq + h * G) * a.score_stride;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < G; ++i) {
    const float z = lse_sm[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + j * 256;
      if (t >= lo && t < ctx) sum[j] += fast_exp2(s[i * a.score_stride + t] - z);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = t0 + j * 256;
    if (t >= lo && t < ctx) atomicAdd(w + t, sum[j]);  // (another sequence may have the slot; its own tokens get one sum each)
  }
}

// Whether pairs are left whole, so that no second kernel has to add their parts up (4 to 7 us), although a CTA may get the tiles of almost
// a pair more than its even share. us, cut / whole, 32 heads of 128: 8 pairs of up to 4 tiles 8.9 / 7.7, of up to 8 8.2 / 10.2; 64 pairs of up to 8
// 11.7 / 11.3, of up to 16 14.0 / 16.4; 1624 pairs of up to 8 47.8 / 44.3, of up to 16 69.7 / 65.4. (Heads of 64 and groups of more than 8 heads
// have the same limits, with other CTAs per SM; there they are right by tests, not by times.)
int most_tiles(int window, int max_ctx) {  // of a pair
  return window > 0 && window < max_ctx ? ceil_div(window - 1, kKeyTile) + 1 : ceil_div(max_ctx, kKeyTile);
}
bool uncut(int64_t pairs, int tiles) { return tiles <= (pairs >= 1024 ? 16 : pairs >= 64 ? 8 : 4); }

// floats of the workspace: partial results, log2 of the sums, scores
struct Layout {
  int64_t lse, scores, score_stride, total;
  int ctas;
  Layout(int B, int Hq, int Hkv, int D, int max_ctx, bool weights) {
    const int64_t tiles = static_cast<int64_t>(B) * Hkv * (ceil_div64(max_ctx, kKeyTile) + 1);
    const int full = ctas_per_sm(D, Hq / Hkv > 8 ? 2 : 1) * pxl_host::num_sms();
    ctas = tiles < full ? static_cast<int>(tiles) : full;
    lse = static_cast<int64_t>(ctas) * 2 * (Hq / Hkv * (D + 2) + 4);
    score_stride = weights ? ceil_div64(max_ctx, kKeyTile) * kKeyTile : 0;
    scores = ceil_div64(lse + (weights ? static_cast<int64_t>(B) * Hq : 0), 32) * 32;
    total = scores + score_stride * B * Hq;
  }
};

// How many CTAs share a pair, as a power of two, so that all pairs are on the chip at once; 0: pairs are dealt out. us, dealt out / eight, four or
// two CTAs, 32 heads of 128 on 8: one sequence of up to 776 tokens 9.9 / 6.9, of up to 6000 19.0 / 12.8, of up to 12000 18.5 / 20.0; 12 of up to
// 1500 16.0 / 12.3 (four), of up to 6000 28.6 / 31.1; 27 of up to 1500 19.5 / 17.3 (two), of up to 6000 47.1 / 51.8.
template <int D, int NH>
int log_ranks_of(int64_t pairs, int tiles) {
  static std::atomic<int> known[64][kLogRanks + 1];  // clusters that are on the chip at once + 1
  for (int log = kLogRanks; log > 0; --log) {
    if (tiles > (log == kLogRanks ? 128 : 32)) continue;
    std::atomic<int>& entry = known[pxl_host::current_device_slot()][log];
    int n = entry.load(std::memory_order_relaxed) - 1;
    if (n < 0) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(1 << log);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = Shape<D, NH>::kSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << log;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, attn_i8_decode_kernel<D, NH, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      entry.store(n + 1, std::memory_order_relaxed);
    }
    if (pairs <= n) return log;
  }
  return 0;
}

template <int D, int NH>
int launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, Args a, int ctas, int tiles, float* weights, int64_t W, int slots,
                  const int* seq_slots, cudaStream_t stream) {
  constexpr int kSmem = Shape<D, NH>::kSmem;
  static std::atomic<bool> configured[64];  // function attributes are per device
  std::atomic<bool>& done = configured[pxl_host::current_device_slot()];
  if (!done.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(attn_i8_decode_kernel<D, NH, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
        cudaFuncSetAttribute(attn_i8_decode_kernel<D, NH, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return PXL_ERR_CUDA;
    done.store(true, std::memory_order_relaxed);
  }
  const int64_t pairs = static_cast<int64_t>(a.B) * a.Hkv;
  if (!a.uncut) a.log_ranks = log_ranks_of<D, NH>(pairs, tiles);
  if (a.log_ranks) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(pairs << a.log_ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << a.log_ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pxl_host::chained() ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, attn_i8_decode_kernel<D, NH, true>, tk, tv, a) != cudaSuccess) {
      cudaGetLastError();
      return PXL_ERR_CUDA;
    }
  } else {
    pxl_host::launch(attn_i8_decode_kernel<D, NH, false>, dim3(ctas), dim3(kThreads), kSmem, stream, tk, tv, a);
    if (ctas > 1 && !a.uncut)
      pxl_host::launch_behind(attn_i8_join_kernel<D>, dim3(ctas - 1), dim3(kJoinThreads), a.Hq / a.Hkv * ctas * 4, stream, a, ctas);
  }
  if (weights)
    pxl_host::launch_behind(attn_i8_weigh_kernel, dim3(static_cast<unsigned>(ceil_div64(a.score_stride, kWeighKeys)), a.Hkv, a.B), dim3(256), 0,
                            stream, a, weights, W, slots, seq_slots);
  return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

}  // namespace

PXL_EXPORT int64_t pxl_attn_i8_decode_workspace(int B, int Hq, int Hkv, int D, int max_ctx, int with_weights) {
  if (B <= 0 || Hkv <= 0 || max_ctx <= 0) return 0;
  return Layout(B, Hq, Hkv, D, max_ctx, with_weights != 0).total * 4;
}

PXL_EXPORT int pxl_attn_i8_decode(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const float* kv_max,
                                  const int* block_tables, const int* ctx_lens, void* out, int64_t out_stride, const float* sinks,
                                  float* weights, int64_t W, int slots, const int* seq_slots, void* workspace, int64_t workspace_bytes, int B,
                                  int Hq, int Hkv, int D, int page, int max_blocks, int64_t num_blocks, float scale, int window, int max_ctx,
                                  int* status, cudaStream_t stream) {
  if (B <= 0) return PXL_OK;
  if ((D != 64 && D != 128) || (page != 16 && page != 32 && page != 64) || Hkv <= 0 || Hq % Hkv || Hq / Hkv < 1 || Hq / Hkv > 16 ||
      !(scale > 0.f) || (q_stride & 7) || (out_stride & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (reinterpret_cast<uintptr_t>(kv_max) & 7) || max_blocks <= 0 || max_ctx <= 0 || max_ctx >= (1 << 30) ||
      window < 0 || window > (1 << 30) || num_blocks <= 0 ||
      num_blocks * Hkv * page >= (1ll << 31))
    return PXL_ERR_INVALID_ARG;
  const Layout at(B, Hq, Hkv, D, max_ctx, weights != nullptr);
  if (!workspace || workspace_bytes < at.total * 4) return PXL_ERR_INVALID_ARG;
  if (Hkv > 65535 || B > 65535) return PXL_ERR_TOO_LARGE;
  CUtensorMap tk, tv;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * Hkv * page;
  if (!pxl_host::make_tmap_codes(&tk, k_cache, rows, D, page) || !pxl_host::make_tmap_codes(&tv, v_cache, rows, D, page))
    return PXL_ERR_TENSORMAP;
  float* ws = static_cast<float*>(workspace);
  const int tiles = most_tiles(window, max_ctx);
  const Args a{static_cast<const bf16*>(q), q_stride, reinterpret_cast<const float2*>(kv_max), block_tables, ctx_lens, static_cast<bf16*>(out),
               out_stride, sinks, ws, weights ? ws + at.lse : nullptr, weights ? ws + at.scores : nullptr, at.score_stride, B, Hq, Hkv, page,
               max_blocks, num_blocks, scale * kLog2e, window, uncut(static_cast<int64_t>(B) * Hkv, tiles), 0, status};
  auto go = [&](auto launch) { return launch(tk, tv, a, at.ctas, tiles, weights, W, slots, seq_slots, stream); };
  if (D == 64) return Hq / Hkv > 8 ? go(launch_decode<64, 2>) : go(launch_decode<64, 1>);
  return Hq / Hkv > 8 ? go(launch_decode<128, 2>) : go(launch_decode<128, 1>);
}
