// Decode attention over keys and values in 8 bits (layout: kv_i8.cu): one query per sequence.
//
// Every CTA gets the same number of tiles of 64 keys of the row of all (sequence, key head) pairs (attention_walk.cuh). A producer warp
// brings the codes by TMA, page by page, and the pages' magnitudes by 8-byte cp.async into the same stage; four consumer warps, two per
// tile, convert the codes where they multiply them (mma.sync, f16) and keep a running maximum, sum and output of the 16 rows of a warp's
// products (the query heads of a key head; rows 8 to 15 are left out where there are at most 8). A score is multiplied by its page's key
// magnitude in fp32. The output is held relative to the largest value magnitude R so far, beside the running maximum: probabilities times
// a page's share of R are what is rounded to f16 (2^-11), with a factor of 2^15 so that they keep their bits down to 2^-29.
// A pair that lies in several CTAs is added up by a second kernel. Where the weights are wanted, the scores go to the workspace (4 bytes
// per query head and key beside 2 D per key head) and a third kernel adds their exponentials once the sums are known.
#include <atomic>

#include "attention_walk.cuh"
#include "common.cuh"
#include "kv_i8.cuh"
#include "pxl_api.h"
#include "tc_issue.cuh"

namespace {
using namespace pxl;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 160;  // four consumer warps and the producer

template <int D, bool HIGH>
struct Shape {
  static constexpr int kTileBytes = kKeyTile * D;                // of K, or of V
  static constexpr int kStages = D == 64 ? 8 : HIGH ? 4 : 6;     // even: a stage belongs to one pair of warps
  static constexpr int kTiles = D / 8;                           // of 8 columns of the output
  static constexpr int kVecs = kTiles * (HIGH ? 4 : 2) / 4;      // 16-byte vectors of a lane's output
  static constexpr int kOffParts = kStages * 2 * kTileBytes;     // [3][kVecs][32] float4
  static constexpr int kOffStats = kOffParts + 3 * kVecs * 512;  // [3][5][32] floats: maxima, sums, R
  static constexpr int kOffMax = kOffStats + 3 * 5 * 128;        // [stages][4] magnitudes of a stage's pages
  static constexpr int kOffBars = kOffMax + kStages * 32;
  static constexpr int kSmem = 1024 + kOffBars + kStages * 16 + 16;
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
  int* status;
};

__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// arrives once the copies that this thread began are there; the barrier counts the arrival
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <int D, bool HIGH>
struct Rows {
  static constexpr int kRows = HIGH ? 2 : 1, kKeys = 32, kSteps = D / 16;
  uint32_t qf[kSteps][4];
  float row_scale[2], o[D / 8][4], m_run[2], l_run[2], r_run;

  // byte offset of 16-byte chunk c of a row of a tile as TMA lays it down
  static __device__ __forceinline__ uint32_t chunk(int row, int c) {
    return D == 128 ? row * 128 + ((c ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  }

  // q: first query head of the key head. Lane t of a quad takes columns D / 4 * t and on, of q as of the keys.
  __device__ __forceinline__ void begin(const bf16* q, int G, float scale_log2) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g8 + h * 8;
      float mx = 0.f;
      if ((HIGH || h == 0) && r < G) {
        const uint2* row = reinterpret_cast<const uint2*>(q + r * D + t4 * (D / 4));
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          const uint2 x = row[ks];
          qf[ks][h] = x.x;
          qf[ks][2 + h] = x.y;
          const float2 a = unpack_bf16x2(x.x), b = unpack_bf16x2(x.y);
          mx = fmaxf(fmaxf(fmaxf(mx, fabsf(a.x)), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y)));
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) qf[ks][h] = qf[ks][2 + h] = 0u;
      }
      if (!HIGH && h == 1) break;
      float down;
      const float up = row_up(quad_max(mx), down);
      row_scale[h] = down * scale_log2 * kInv127;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float2 x = unpack_bf16x2(qf[ks][2 * p + h]);
          qf[ks][2 * p + h] = pack_f16x2(x.x * up, x.y * up);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m_run[0] = m_run[1] = -INFINITY;
    l_run[0] = l_run[1] = r_run = 0.f;
  }

  // Keys r0 .. r0 + 31 of a tile; the first is token tok_base. near, far: magnitudes of the pages of its first and second 16. scores: where
  // they go for row 0 of the pair (null: nowhere), a row `score_stride` behind the one before.
  __device__ __forceinline__ void step(uint32_t k_smem, uint32_t v_smem, int r0, int tok_base, int lo, int hi, float2 near, float2 far,
                                       float* scores, int64_t score_stride, int G) {
    if (!(tok_base < hi && tok_base + kKeys > lo)) return;  // warp-uniform
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    float s[4][4];  // 8 tokens each
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
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
        for (int j = 0; j < 4; ++j) {
          const uint32_t f = flip_codes(w[j][i]);
          mma_m16n8k16_f16(s[j], qf[c * 4 + i], codes_f16x2<0x4140>(f), codes_f16x2<0x4342>(f));
        }
    }
    const bool whole = tok_base + kKeys <= hi && tok_base >= lo;  // every token is seen
    float corr[2] = {1.f, 1.f};
    // (of pages that have a token which is seen; a NaN is passed over)
    const float r_new = fmaxf(r_run, fmaxf(tok_base + 16 > lo ? near.y : 0.f, tok_base + 16 < hi ? far.y : 0.f));
    const float share[2] = {page_share(near.y, r_new), page_share(far.y, r_new)};
    const float r_corr = r_new > r_run ? page_share(r_run, r_new) : 1.f;
    r_run = r_new;
#pragma unroll
    for (int h = 0; h < kRows; ++h) {
      const float scale[2] = {row_scale[h] * near.x, row_scale[h] * far.x};
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 2 * h; e < 2 * h + 2; ++e) {
          s[j][e] *= scale[j >> 1];
          if (!whole) {
            const int tok = tok_base + j * 8 + 2 * t4 + (e & 1);
            if (!(tok < hi && tok >= lo)) s[j][e] = -INFINITY;
          }
          mx = fmaxf(mx, s[j][e]);
        }
      if (scores && g8 + 8 * h < G) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float2*>(scores + (g8 + 8 * h) * score_stride + tok_base + j * 8 + 2 * t4) = make_float2(s[j][2 * h], s[j][2 * h + 1]);
      }
      const float m_new = fmaxf(m_run[h], quad_max(mx));
      const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
      corr[h] = fast_exp2(m_run[h] - m_use);
      m_run[h] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 2 * h; e < 2 * h + 2; ++e) {
          const float p = fast_exp2(s[j][e] - m_use + kPUp);
          ps += p;
          s[j][e] = whole || s[j][e] != -INFINITY ? p * share[j >> 1] : 0.f;  // (a share that is NaN, of a token that is not seen)
        }
      l_run[h] = l_run[h] * corr[h] + ps;
      corr[h] *= r_corr;
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || (HIGH && corr[1] != 1.f))) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2 * kRows; ++e) o[i][e] *= corr[e >> 1];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t pf[4];
      pf[0] = pack_f16x2(s[2 * k][0], s[2 * k][1]);
      pf[1] = HIGH ? pack_f16x2(s[2 * k][2], s[2 * k][3]) : 0u;
      pf[2] = pack_f16x2(s[2 * k + 1][0], s[2 * k + 1][1]);
      pf[3] = HIGH ? pack_f16x2(s[2 * k + 1][2], s[2 * k + 1][3]) : 0u;
      const int mi = lane >> 3, row = r0 + k * 16 + (mi & 1) * 8 + (lane & 7);
#pragma unroll
      for (int c = 0; c < D / 16; c += 2) {  // 16 columns per chunk; a transposed pair of bytes is two columns of a token
        uint32_t r[4];                       // chunk c: tokens 0-7, 8-15; chunk c + 1: the same
        ldmatrix_x4_trans(r, v_smem + chunk(row, c + (mi >> 1)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a = flip_codes(r[2 * h]), b = flip_codes(r[2 * h + 1]);
          mma_m16n8k16_f16(o[(c + h) * 2], pf, codes_f16x2<0x4240>(a), codes_f16x2<0x4240>(b));          // even columns
          mma_m16n8k16_f16(o[(c + h) * 2 + 1], pf, codes_f16x2<0x4341>(a), codes_f16x2<0x4341>(b));      // odd ones
        }
      }
    }
  }

  // columns of o[i][2 r], o[i + 1][2 r], o[i][2 r + 1], o[i + 1][2 r + 1] (i even): four in a row
  static __device__ __forceinline__ int column(int i) { return i * 8 + 4 * (threadIdx.x & 3); }
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
// 1 / sum in units of R, and log2 of the sum of exponentials, for a row with a sink or without
__device__ __forceinline__ float finish(float M, float L, float R, float sink, float& lse) {
  const float Mx = fmaxf(M, sink), Mu = Mx == -INFINITY ? 0.f : Mx;
  const float e = fast_exp2(M - Mu), denom = L * e + fast_exp2(sink - Mu + kPUp);
  lse = denom == 0.f ? INFINITY : Mu + log2f(denom) - kPUp;
  return denom == 0.f ? 0.f : e / denom * (R * kInv127);
}

template <int D, bool HIGH>
__global__ void __launch_bounds__(kThreads, 2)
attn_i8_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using S = Shape<D, HIGH>;
  using R = Rows<D, HIGH>;
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
  DecodeWalk walk(work, blockIdx.x, gridDim.x);
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

      // warps 2 and 3 hand their results to 0 and 1, 1 to 0; a register goes to the same lane
      auto give = [&](int p) {
#pragma unroll
        for (int i = 0; i < S::kVecs; ++i) {
          if constexpr (HIGH) parts[(p * S::kVecs + i) * 32 + lane] = make_float4(rows.o[i][0], rows.o[i][1], rows.o[i][2], rows.o[i][3]);
          else parts[(p * S::kVecs + i) * 32 + lane] = make_float4(rows.o[2 * i][0], rows.o[2 * i][1], rows.o[2 * i + 1][0], rows.o[2 * i + 1][1]);
        }
        float* st = stats + p * 5 * 32 + lane;
        st[0] = rows.m_run[0], st[32] = rows.l_run[0], st[64] = rows.m_run[1], st[96] = rows.l_run[1], st[128] = rows.r_run;
      };
      auto add = [&](int p) {
        const float* st = stats + p * 5 * 32 + lane;
        const float r_new = fmaxf(rows.r_run, st[128]);
        const Joined x(rows.m_run[0], rows.l_run[0], rows.r_run, r_new, st[0], st[32], st[128]);
        if constexpr (HIGH) {
          const Joined y(rows.m_run[1], rows.l_run[1], rows.r_run, r_new, st[64], st[96], st[128]);
#pragma unroll
          for (int i = 0; i < S::kVecs; ++i) {
            const float4 v = parts[(p * S::kVecs + i) * 32 + lane];
            rows.o[i][0] = rows.o[i][0] * x.fa + v.x * x.fb;
            rows.o[i][1] = rows.o[i][1] * x.fa + v.y * x.fb;
            rows.o[i][2] = rows.o[i][2] * y.fa + v.z * y.fb;
            rows.o[i][3] = rows.o[i][3] * y.fa + v.w * y.fb;
          }
        } else {
#pragma unroll
          for (int i = 0; i < S::kVecs; ++i) {
            const float4 v = parts[(p * S::kVecs + i) * 32 + lane];
            rows.o[2 * i][0] = rows.o[2 * i][0] * x.fa + v.x * x.fb;
            rows.o[2 * i][1] = rows.o[2 * i][1] * x.fa + v.y * x.fb;
            rows.o[2 * i + 1][0] = rows.o[2 * i + 1][0] * x.fa + v.z * x.fb;
            rows.o[2 * i + 1][1] = rows.o[2 * i + 1][1] * x.fa + v.w * x.fb;
          }
        }
        rows.r_run = r_new;
      };
      if (warp >= 2) give(warp - 2);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (warp < 2) add(warp);
      if (warp == 1) give(2);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (warp == 0) {
        add(2);
#pragma unroll
        for (int h = 0; h < (HIGH ? 2 : 1); ++h) {
          const int r = (lane >> 2) + 8 * h;
          const float M = rows.m_run[h], L = quad_sum(rows.l_run[h]);
          if (r >= G || failed) continue;
          if (walk.whole()) {
            float lse;
            const float f = finish(M, L, rows.r_run, a.sinks ? a.sinks[head0 + r] * kLog2e : -INFINITY, lse);
            if (a.lse && (lane & 3) == 0) a.lse[static_cast<size_t>(walk.b) * a.Hq + head0 + r] = lse;
            bf16* dst = a.out + walk.b * a.out_stride + (head0 + r) * D;
#pragma unroll
            for (int i = 0; i < D / 8; i += 2)
              *reinterpret_cast<uint2*>(dst + R::column(i)) = make_uint2(pack_bf16x2(rows.o[i][2 * h] * f, rows.o[i + 1][2 * h] * f),
                                                                         pack_bf16x2(rows.o[i][2 * h + 1] * f, rows.o[i + 1][2 * h + 1] * f));
          } else {
            float* po = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (walk.t == 0 ? 1 : 0)) * (G * (D + 2) + 4);
#pragma unroll
            for (int i = 0; i < D / 8; i += 2) {
              float* at = po + r * D + R::column(i);
              at[0] = rows.o[i][2 * h], at[1] = rows.o[i + 1][2 * h], at[2] = rows.o[i][2 * h + 1], at[3] = rows.o[i + 1][2 * h + 1];
            }
            if ((lane & 3) == 0) po[G * D + r] = M, po[G * D + G + r] = L, po[G * (D + 2)] = rows.r_run;
          }
        }
      }
    }
  }
  if (__syncthreads_or(failed)) __nanosleep(200000);  // loads that are still in flight must land before the shared memory is released
}

// Adds up the pairs that lie in several CTAs. Block x: the pair that the border between CTAs x and x + 1 cuts, if no border before it does.
template <int D>
__global__ void __launch_bounds__(D)
attn_i8_join_kernel(const __grid_constant__ Args a, int ctas) {
  constexpr int R = 4;  // query heads at a time, so that their loads are in flight together
  const DecodeWork work{a.ctx_lens, a.B, a.Hkv, a.window, 0};
  const int cut = blockIdx.x + 1, d = threadIdx.x, G = a.Hq / a.Hkv;
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
  const size_t place = static_cast<size_t>(G) * (D + 2) + 4;
  auto part = [&](int x) { return a.parts + (static_cast<size_t>(x) * 2 + (x < cut ? 1 : 0)) * place; };
  float r_all = 0.f;
  for (int x = cut - 1; x <= last; ++x) r_all = fmaxf(r_all, part(x)[G * (D + 2)]);
  for (int r0 = 0; r0 < G; r0 += R) {
    float acc[R], L[R], M[R];
#pragma unroll
    for (int i = 0; i < R; ++i) acc[i] = L[i] = 0.f, M[i] = -INFINITY;
    for (int x = cut - 1; x <= last; ++x) {
      const float* p = part(x) + r0 * D + d;
      const float *pm = part(x) + G * D + r0, *pl = pm + G;
      const float rx = part(x)[G * (D + 2)];
      float o[R], m[R], l[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const bool in = r0 + i < G;
        o[i] = in ? p[i * D] : 0.f;
        m[i] = in ? pm[i] : -INFINITY;
        l[i] = in ? pl[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const Joined f(M[i], L[i], r_all, r_all, m[i], l[i], rx);
        acc[i] = acc[i] * f.fa + o[i] * f.fb;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i >= G) break;
      const int head = kvh * G + r0 + i;
      float lse;
      const float f = finish(M[i], L[i], r_all, a.sinks ? a.sinks[head] * kLog2e : -INFINITY, lse);
      if (a.lse && d == 0) a.lse[static_cast<size_t>(b) * a.Hq + head] = lse;
      a.out[b * a.out_stride + head * D + d] = __float2bfloat16(acc[i] * f);
    }
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
    if (t >= lo && t < ctx) w[t] += sum[j];
  }
}

// floats of the workspace: partial results, log2 of the sums, scores
struct Layout {
  int64_t lse, scores, score_stride, total;
  int ctas;
  Layout(int B, int Hq, int Hkv, int D, int max_ctx, bool weights) {
    const int64_t tiles = static_cast<int64_t>(B) * Hkv * (ceil_div64(max_ctx, kKeyTile) + 1);
    const int full = 2 * pxl_host::num_sms();
    ctas = tiles < full ? static_cast<int>(tiles) : full;
    lse = static_cast<int64_t>(ctas) * 2 * (Hq / Hkv * (D + 2) + 4);
    score_stride = weights ? ceil_div64(max_ctx, kKeyTile) * kKeyTile : 0;
    scores = ceil_div64(lse + (weights ? static_cast<int64_t>(B) * Hq : 0), 32) * 32;
    total = scores + score_stride * B * Hq;
  }
};

template <int D, bool HIGH>
int launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int ctas, float* weights, int64_t W, int slots,
                  const int* seq_slots, cudaStream_t stream) {
  constexpr int kSmem = Shape<D, HIGH>::kSmem;
  static std::atomic<bool> configured[64];  // function attributes are per device
  std::atomic<bool>& done = configured[pxl_host::current_device_slot()];
  if (!done.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(attn_i8_decode_kernel<D, HIGH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return PXL_ERR_CUDA;
    done.store(true, std::memory_order_relaxed);
  }
  pxl_host::launch(attn_i8_decode_kernel<D, HIGH>, dim3(ctas), dim3(kThreads), kSmem, stream, tk, tv, a);
  if (ctas > 1) pxl_host::launch_behind(attn_i8_join_kernel<D>, dim3(ctas - 1), dim3(D), 0, stream, a, ctas);
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
      (reinterpret_cast<uintptr_t>(kv_max) & 7) || max_blocks <= 0 || max_ctx <= 0 || window < 0 || num_blocks <= 0 ||
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
  const Args a{static_cast<const bf16*>(q), q_stride, reinterpret_cast<const float2*>(kv_max), block_tables, ctx_lens, static_cast<bf16*>(out),
               out_stride, sinks, ws, weights ? ws + at.lse : nullptr, weights ? ws + at.scores : nullptr, at.score_stride, B, Hq, Hkv, page,
               max_blocks, num_blocks, scale * kLog2e, window, status};
  auto go = [&](auto launch) { return launch(tk, tv, a, at.ctas, weights, W, slots, seq_slots, stream); };
  if (D == 64) return Hq / Hkv > 8 ? go(launch_decode<64, true>) : go(launch_decode<64, false>);
  return Hq / Hkv > 8 ? go(launch_decode<128, true>) : go(launch_decode<128, false>);
}
