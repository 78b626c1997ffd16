// Products of bf16 rows with microscaled 4-bit weights on the 5th-generation tensor cores:
//
//   C[t, n] = row_scale[n] * sum_k x[t, k] * v[n, k] (+ bias[n]) (+ residual[t, n]),  or gated
//
// e2m1 numbers times powers of two are exact in bf16, so that the product is that of the expanded weights; they are expanded on
// their way from shared to tensor memory. The weights take the operand that tensor memory can hold (128 rows of them per tile), the
// rows of x the other (N of the instruction, 16 to 256), so that a few rows cost a few columns and accumulators are [n][t].
//
// Warps of a CTA: 0 loads (a block of weights is one bulk copy, rows of x come by TMA), 1 issues, 2-5 write results, 6-13 expand.
// A thread of the latter has one weight row: 64 codes per block of 128 columns, eight at a time from a 32-bit word into four bf16
// pairs, stored to tensor memory as the instruction's A operand.
#include "common.cuh"
#include "mx4.cuh"
#include "pxl_api.h"
#include "tc_issue.cuh"

namespace {
using namespace pxl;

constexpr int kWarps = 14, kThreads = kWarps * 32;
constexpr int kWeightBytes = 9216;        // a block of weights in a stage, filled up to 1024 bytes
constexpr int kPitch = kTileRows + 4;     // floats of a token's results in shared memory
constexpr int kChunk = 32;                // tokens whose results are staged at a time
constexpr int kStaging = kChunk * kPitch * 4;
constexpr int kMaxStages = 8;
constexpr int kMaxExperts = 1024;

struct TcArgs {
  const uint8_t* w;
  const float* row_scale;
  void* C;
  const bf16* bias;
  const bf16* residual;
  int64_t ldc, ldr;
  int M, N, epi, out_f32;
  float limit;
  int n_blocks, k_blocks, t_tiles;
  int bt, box;           // tokens of a tile (a multiple of 16) and of a TMA box
  int stages, a_bufs, d_bufs, d_cols;
  int splits, kb_per;    // SPLIT: CTAs of a cluster, one per range of K blocks
  const int* offsets;    // grouped: first row of every expert, and the end
  int experts;
  int vec;               // results and residual in whole 16-byte vectors
  int early;             // in a launch chain: the first weights are read ahead of the wait
};

struct Item {
  int n_blk, row0, rows, expert;
};

// Item i of the launch: a block of weight rows, and a tile of tokens. Tiles of tokens follow one another for a block of weights,
// unless there are experts: then the blocks of an expert's weights follow for a tile.
__device__ __forceinline__ Item item_of(int i, const TcArgs& g, const int* first_tile) {
  Item it;
  if (g.offsets == nullptr) {
    it.n_blk = i / g.t_tiles;
    it.row0 = (i % g.t_tiles) * g.bt;
    it.rows = min(g.bt, g.M - it.row0);
    it.expert = 0;
    return it;
  }
  const int tile = i / g.n_blocks;
  it.n_blk = i % g.n_blocks;
  int lo = 0, hi = g.experts;  // the last expert whose first tile is not behind `tile`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= tile) lo = mid;
    else hi = mid;
  }
  it.expert = lo;
  it.row0 = g.offsets[lo] + (tile - first_tile[lo]) * g.bt;
  it.rows = min(g.bt, g.offsets[lo + 1] - it.row0);
  return it;
}

// Eight results of a token: columns c .. c + 7 of the block (of its 64 outputs, where it is gated).
__device__ __forceinline__ void finish8(const TcArgs& g, float (&f)[16], bool glu, int n_blk, int t, int c) {
  const int n0 = n_blk * (glu ? 64 : 128) + c, n_out = glu ? g.N / 2 : g.N;
  if (n0 >= n_out) return;
  if (glu) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = mx4_gate(f[j], f[8 + j], g.epi, g.limit);
  }
  const bool whole = g.vec && n0 + 8 <= n_out;
  if (g.residual) {
    const bf16* r = g.residual + t * g.ldr + n0;
    if (whole) {
      const bf16x8 v = ld_bf16x8(r);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 p = unpack_bf16x2(v.u[j]);
        f[2 * j] += p.x, f[2 * j + 1] += p.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n0 + j < n_out) f[j] += __bfloat162float(r[j]);
    }
  }
  if (g.out_f32) {
    float* dst = static_cast<float*>(g.C) + t * g.ldc + n0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n0 + j < n_out) dst[j] = f[j];
    return;
  }
  bf16* dst = static_cast<bf16*>(g.C) + t * g.ldc + n0;
  if (whole) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.u[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
    st_bf16x8(dst, o);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n0 + j < n_out) dst[j] = __float2bfloat16(f[j]);
  }
}

template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmap, const TcArgs g, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stage_bytes = kWeightBytes + g.bt * 256;
  float* staging = reinterpret_cast<float*>(smem + g.stages * stage_bytes);
  int* first_tile = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(staging) + (SPLIT ? 0 : kStaging));
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * 4 + 2 * 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, afull0 = empty0 + 8 * kMaxStages, aempty0 = afull0 + 32,
                 dfull0 = aempty0 + 32, dempty0 = dfull0 + 16;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int tmem_cols = g.d_bufs * g.d_cols + g.a_bufs * 64 > 256 ? 512 : 256;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < g.stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int b = 0; b < g.a_bufs; ++b) mbar_init(afull0 + 8 * b, 8), mbar_init(aempty0 + 8 * b, 1);
    for (int b = 0; b < g.d_bufs; ++b) mbar_init(dfull0 + 8 * b, 1), mbar_init(dempty0 + 8 * b, 4);
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmap);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  int items = g.n_blocks * g.t_tiles;
  if (g.offsets != nullptr) {
    pdl_wait();  // the experts' rows come from the kernels before
    if (warp == 0) {
      int sum = 0;
      for (int e0 = 0; e0 < g.experts; e0 += 32) {
        const int e = e0 + lane;
        int n = e < g.experts ? ceil_div(g.offsets[e + 1] - g.offsets[e], g.bt) : 0;
        const int own = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, n, o);
          if (lane >= o) n += a;
        }
        if (e < g.experts) first_tile[e] = sum + n - own;
        sum += __shfl_sync(0xffffffffu, n, 31);
      }
      if (lane == 0) first_tile[g.experts] = sum;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot, tmem_a = tmem + g.d_bufs * g.d_cols;
  if (g.offsets != nullptr) items = first_tile[g.experts] * g.n_blocks;

  const int i0 = SPLIT ? blockIdx.x / g.splits : blockIdx.x, i_step = SPLIT ? items : gridDim.x;
  const int kb0 = SPLIT ? static_cast<int>(cluster_cta_rank()) * g.kb_per : 0;
  const int kb1 = SPLIT ? min(kb0 + g.kb_per, g.k_blocks) : g.k_blocks;
  auto weights = [&](const Item& it, int kb) {
    return g.w + ((static_cast<int64_t>(it.expert) * g.n_blocks + it.n_blk) * g.k_blocks + kb) * kBlockBytes;
  };
  auto stage_tx = [&](const Item& it) { return static_cast<uint32_t>(kBlockBytes + ceil_div(it.rows, g.box) * g.box * 256); };

  const bool early = g.early && i0 < items;  // (never with experts, whose lists are written in the chain)
  if (warp == 0 && lane == 0 && early) {
    const Item it = item_of(i0, g, first_tile);
    for (int s = 0; s < g.stages && kb0 + s < kb1; ++s) {
      mbar_arrive_expect_tx(full0 + 8 * s, stage_tx(it));
      bulk_load_g2s(smem_u32(smem + s * stage_bytes), weights(it, kb0 + s), kBlockBytes, full0 + 8 * s);
    }
  }
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    const uint32_t leader = elect_leader(), s0 = smem_u32(smem);
    int stage = 0, done = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, first_tile);
      const int boxes = ceil_div(it.rows, g.box);
      for (int kb = kb0; kb < kb1; ++kb, ++done) {
        const uint32_t fb = full0 + 8 * stage, at = s0 + stage * stage_bytes;
        if (!early || done >= g.stages) {
          ok = wait_warp(empty0 + 8 * stage, phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          expect_tx(fb, stage_tx(it), leader);
          if (leader) bulk_load_g2s(at, weights(it, kb), kBlockBytes, fb);
        }
        for (int b = 0; b < boxes; ++b) {
          const uint32_t dst = at + kWeightBytes + b * g.box * 128;
          tma_box(dst, &tmap, fb, kb * kTileCols, it.row0 + b * g.box, leader);
          tma_box(dst + g.bt * 128, &tmap, fb, kb * kTileCols + 64, it.row0 + b * g.box, leader);
        }
        if (++stage == g.stages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    int stage = 0, ab = 0, db = 0;
    uint32_t phase = 0, a_phase = 0, d_phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, first_tile);
      const uint32_t idesc = umma_idesc(kTileRows, ceil_div(it.rows, 16) * 16, 1, 1);
      ok = wait_warp(dempty0 + 8 * db, d_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
      for (int kb = kb0; ok && kb < kb1; ++kb) {
        ok = wait_warp(full0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL) &&
             wait_warp(afull0 + 8 * ab, a_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t desc = umma_desc_k_sw128(smem_u32(smem) + stage * stage_bytes + kWeightBytes);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_ts(tmem + db * g.d_cols, tmem_a + ab * 64 + k * 8, desc + ((k >> 2) * g.bt * 8 + (k & 3) * 2), idesc,
                 kb > kb0 || k > 0 ? 1u : 0u, leader);
        commit(empty0 + 8 * stage, leader);
        commit(aempty0 + 8 * ab, leader);
        if (++stage == g.stages) stage = 0, phase ^= 1;
        if (++ab == g.a_bufs) ab = 0, a_phase ^= 1;
      }
      if (!ok) break;
      commit(dfull0 + 8 * db, leader);
      if (++db == g.d_bufs) db = 0, d_phase ^= 1;
    }
  } else if (warp < 6) {
    // ---- results: lane = weight row, columns = tokens; staged in shared memory to be written along the weight rows
    const int q = warp & 3, r = q * 32 + lane, tid = threadIdx.x - 64;
    const bool glu = g.epi != PXL_EPI_NONE;
    int db = 0;
    uint32_t d_phase = 0;
    bool ok = true;
    for (int i = i0; i < items; i += i_step) {
      const Item it = item_of(i, g, first_tile);
      const int n = it.n_blk * kTileRows + r;
      const float factor = g.row_scale[it.expert * g.n_blocks * kTileRows + n];
      const float add = g.bias && n < g.N && kb0 == 0 ? __bfloat162float(g.bias[it.expert * g.N + n]) : 0.f;
      // after a wait that ran out the loop goes on without results: the warps meet at every barrier below
      ok = ok && wait_warp(dfull0 + 8 * db, d_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_FULL);
      tc_fence_after_sync();
      for (int c0 = 0; c0 < it.rows; c0 += kChunk) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem + db * g.d_cols + c0 + (static_cast<uint32_t>(q * 32) << 16), v);
        tmem_ld_wait();
        if (c0 + kChunk >= it.rows) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(dempty0 + 8 * db);
        }
        float* part = SPLIT ? reinterpret_cast<float*>(smem) + c0 * kPitch : staging;
        const int m = min(kChunk, it.rows - c0);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < m) part[j * kPitch + r] = __uint_as_float(v[j]) * factor + add;
        if constexpr (!SPLIT) {
          named_bar_sync(1, 128);
          const int per = glu ? 8 : 16;
          for (int e = tid; e < m * per; e += 128) {
            const int t = e / per, c = e % per * 8;
            float f[16];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              if (h >= 2 && !glu) break;
              const float4 x = *reinterpret_cast<const float4*>(part + t * kPitch + c + (h & 1) * 4 + (h >> 1) * 64);
              f[4 * h] = x.x, f[4 * h + 1] = x.y, f[4 * h + 2] = x.z, f[4 * h + 3] = x.w;
            }
            if (ok) finish8(g, f, glu, it.n_blk, it.row0 + c0 + t, c);
          }
          named_bar_sync(1, 128);
        }
      }
      if (++db == g.d_bufs) db = 0, d_phase ^= 1;
    }
  } else {
    // ---- codes -> bf16 in tensor memory
    const int q = warp & 3, half = (warp - 6) >> 2, r = q * 32 + lane;
    const uint32_t row_at = smem_u32(smem) + half * 2 * (kTileRows * 16) + r * 16, pow_at = smem_u32(smem) + kCodeBytes + r * 4;
    const uint32_t dst0 = tmem_a + half * 32 + (static_cast<uint32_t>(q * 32) << 16);
    int stage = 0, ab = 0;
    uint32_t phase = 0, a_phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = wait_warp(full0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL);
        if (!ok) break;
        uint32_t w[2][4], p;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[h][0]), "=r"(w[h][1]), "=r"(w[h][2]), "=r"(w[h][3])
                       : "r"(row_at + stage * stage_bytes + h * (kTileRows * 16)));
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(p) : "r"(pow_at + stage * stage_bytes));
        p >>= half * 16;
        ok = wait_warp(aempty0 + 8 * ab, a_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t p2 = mx4_power2((p >> (8 * h)) & 255u);
          uint32_t o[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t y[4];
            mx4_word(w[h][j], p2, y);
#pragma unroll
            for (int v = 0; v < 4; ++v) o[4 * j + v] = y[v];
          }
          tmem_st_32x32b_x16(dst0 + ab * 64 + h * 16, o);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(afull0 + 8 * ab);
        if (++stage == g.stages) stage = 0, phase ^= 1;
        if (++ab == g.a_bufs) ab = 0, a_phase ^= 1;
      }
    }
  }

  if constexpr (SPLIT) {
    // Every thread of every CTA passes both barriers, also after a failed wait (all other waits are bounded). Between them CTA r
    // adds its share of the tile's tokens over the cluster, in K order, and writes it.
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2) {
      const Item it = item_of(i0, g, first_tile);
      const int share = ceil_div(it.rows, g.splits), r0 = static_cast<int>(cluster_cta_rank()) * share, r1 = min(r0 + share, it.rows);
      const bool glu = g.epi != PXL_EPI_NONE;
      const int per = glu ? 8 : 16;
      for (int e = static_cast<int>(threadIdx.x) - 64; e < (r1 - r0) * per; e += kThreads - 64) {
        const int t = r0 + e / per, c = e % per * 8;
        float f[16] = {};
        for (int s = 0; s < g.splits; ++s) {
          const uint32_t src = cluster_map_shared(smem_u32(smem) + (t * kPitch + c) * 4, s);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            if (h >= 2 && !glu) break;
            const float4 x = ld_shared_cluster_f32x4(src + (h & 1) * 16 + (h >> 1) * 256);
            f[4 * h] += x.x, f[4 * h + 1] += x.y, f[4 * h + 2] += x.z, f[4 * h + 3] += x.w;
          }
        }
        if (!*abort_flag) finish8(g, f, glu, it.n_blk, it.row0 + t, c);
      }
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are being read
  }
  __syncwarp();
  if (*abort_flag) __nanosleep(200000);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, tmem_cols);
}

int launch_tc(const void* x, int64_t ldx, uint64_t x_rows, int K, TcArgs g, int items, int* status, cudaStream_t stream) {
  const int sms = pxl_host::num_sms();
  // two CTAs per SM where their tiles are narrow: 256 columns of tensor memory and half of the shared memory each
  const bool two = g.bt <= 128;
  g.a_bufs = two ? 2 : 4;
  g.d_bufs = 1;
  g.d_cols = pxl::ceil_div(g.bt, 32) * 32;
  const int stage_bytes = kWeightBytes + g.bt * 256, lists = g.offsets ? (g.experts + 1) * 4 : 0;
  const int slots = two ? 2 * sms : sms;
  g.splits = 1;
  if (!g.offsets) {
    int s = slots / items;
    s = s > 8 ? 8 : s;
    while (s > 1 && g.k_blocks / s < 2) --s;
    if (s > 1) {
      g.kb_per = pxl::ceil_div(g.k_blocks, s);
      g.splits = pxl::ceil_div(g.k_blocks, g.kb_per);  // (no empty range)
    }
  }
  const int budget = (two ? 113 : 226) * 1024 - 1024 - 512 - lists - (g.splits > 1 ? 0 : kStaging);
  g.stages = budget / stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  if (g.stages < 1) return PXL_ERR_TOO_LARGE;
  int smem = 1024 + g.stages * stage_bytes + lists + (g.splits > 1 ? 0 : kStaging);
  if (g.splits > 1 && g.stages * stage_bytes < g.bt * kPitch * 4) smem = 1024 + g.bt * kPitch * 4;
  CUtensorMap tmap;
  if (!pxl_host::make_tmap_2d(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, x_rows, K, ldx, g.box, 64)) return PXL_ERR_TENSORMAP;
  static bool configured[64] = {false};
  const int dev = pxl_host::current_device_slot();
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(gemm_mx4_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess ||
        cudaFuncSetAttribute(gemm_mx4_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess)
      return PXL_ERR_CUDA;
    configured[dev] = true;
  }
  if (g.splits > 1) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(items * g.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(g.splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    g.early = pxl_host::chained();
    cfg.numAttrs = g.early ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, gemm_mx4_kernel<true>, tmap, g, status) == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
  }
  g.early = !g.offsets && pxl_host::launch_chain() == pxl_host::kInChain;
  pxl_host::launch(gemm_mx4_kernel<false>, items < slots ? items : slots, kThreads, smem, stream, tmap, g, status);
  return cudaGetLastError() == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

bool epi_known(int epi, int N) {
  return epi == PXL_EPI_NONE || ((epi == PXL_EPI_SILU_MUL || epi == PXL_EPI_CLIP_GLU) && N % 128 == 0);
}
bool on16(const void* p, int64_t ld) { return !((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * 2)) & 15); }

}  // namespace

PXL_EXPORT int pxl_gemm_mx4(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc,
                            const void* bias, const void* residual, int64_t ldr, int M, int N, int K, int epi, float limit,
                            int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 || !epi_known(epi, N) || !on16(x, ldx)) return PXL_ERR_INVALID_ARG;
  TcArgs g{};
  g.w = static_cast<const uint8_t*>(w), g.row_scale = row_scale, g.C = C, g.ldc = ldc;
  g.bias = static_cast<const bf16*>(bias), g.residual = static_cast<const bf16*>(residual), g.ldr = ldr;
  g.M = M, g.N = N, g.epi = epi, g.limit = limit;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kTileCols);
  g.t_tiles = pxl::ceil_div(M, 256);
  g.bt = pxl::ceil_div(pxl::ceil_div(M, g.t_tiles), 16) * 16;
  g.box = g.bt;
  g.vec = on16(C, ldc) && (!residual || on16(residual, ldr));
  return launch_tc(x, ldx, M, K, g, g.n_blocks * g.t_tiles, status, stream);
}

PXL_EXPORT int pxl_gemm_mx4_grouped(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc,
                                    int out_f32, const void* bias, int P, int E, int N, int K, const int* offsets, int epi,
                                    float limit, int* status, cudaStream_t stream) {
  if (P <= 0 || E <= 0 || E > kMaxExperts || N <= 0 || K <= 0 || K % 32 || !epi_known(epi, N) || !on16(x, ldx)) return PXL_ERR_INVALID_ARG;
  TcArgs g{};
  g.w = static_cast<const uint8_t*>(w), g.row_scale = row_scale, g.C = C, g.ldc = ldc, g.out_f32 = out_f32;
  g.bias = static_cast<const bf16*>(bias), g.M = P, g.N = N, g.epi = epi, g.limit = limit;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kTileCols);
  g.offsets = offsets, g.experts = E;
  const int mean = pxl::ceil_div(P, E);
  g.bt = mean <= 16 ? 32 : mean <= 64 ? 64 : mean <= 256 ? 128 : 256;
  g.box = g.bt < 32 ? g.bt : 32;
  g.vec = !out_f32 && on16(C, ldc);
  const int64_t items = static_cast<int64_t>(g.n_blocks) * (pxl::ceil_div(P, g.bt) + (P < E ? P : E));  // at most
  return launch_tc(x, ldx, P, K, g, static_cast<int>(items > 0x7fffffff ? 0x7fffffff : items), status, stream);
}
