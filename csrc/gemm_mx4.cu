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
//
// What bounds it, with the rows of x. Up to 64: the expansion, 15 instructions per word, of two CTAs per SM: 13 x 51200 x 5120 takes 39 us,
// 3.6 TB/s of weights (issue slots 67 % full, tensor pipe 11 %). 65 to 256: the bytes of x that every block of weights needs once more, through
// the SM's port: 203 x 5120 x 25600 60 us, 0.9 PFLOP/s. More: the products, 8192 x 24576 x 4096 1.31 ms, 1.25 PFLOP/s under the power cap.
#include "mx4_tile.cuh"

namespace {
using namespace pxl;

constexpr int kSets = 2, kThreads = (6 + 4 * kSets) * 32;
constexpr int kMaxBufs = 4;
constexpr int kWeightBytes = 9216;  // a block of weights in a stage, filled up to 1024 bytes
constexpr int kMaxStages = 8;
constexpr int kMaxExperts = 1024;

template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmap, const uint8_t* __restrict__ w,
                                                                int a_bufs, const Mx4Shift shift, int* status, const TileArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stage_bytes = kWeightBytes + g.bt * 256;
  float* staging = reinterpret_cast<float*>(smem + g.stages * stage_bytes);
  int* first_tile = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(staging) + (!SPLIT && g.epi != PXL_EPI_NONE ? kStaging : 0));
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kMaxBufs + 2 * 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, afull0 = empty0 + 8 * kMaxStages, aempty0 = afull0 + 8 * kMaxBufs,
                 dfull0 = aempty0 + 8 * kMaxBufs, dempty0 = dfull0 + 16;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int tmem_cols = g.d_bufs * g.d_cols + a_bufs * 64 > 256 ? 512 : 256;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < g.stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int b = 0; b < a_bufs; ++b) mbar_init(afull0 + 8 * b, 4), mbar_init(aempty0 + 8 * b, 1);
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
    return w + ((static_cast<int64_t>(it.expert) * g.n_blocks + it.n_blk) * g.k_blocks + kb) * kBlockBytes;
  };
  const uint32_t stage_tx = kBlockBytes + g.bt * 256;

  // blocks whose weights are read ahead: of the first tile (never with experts, whose lists are written in the chain)
  const int ahead = g.early && i0 < items ? min(g.stages, kb1 - kb0) : 0;
  if (warp == 0 && lane == 0 && ahead > 0) {
    const Item it = item_of(i0, g, first_tile);
    for (int s = 0; s < ahead; ++s) {
      mbar_arrive_expect_tx(full0 + 8 * s, stage_tx);
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
      for (int kb = kb0; kb < kb1; ++kb, ++done) {
        const uint32_t fb = full0 + 8 * stage, at = s0 + stage * stage_bytes;
        if (done >= ahead) {
          ok = wait_parked(empty0 + 8 * stage, phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          expect_tx(fb, stage_tx, leader);
          if (leader) bulk_load_g2s(at, weights(it, kb), kBlockBytes, fb);
        }
        // (rows behind an expert's last one come along: less costly than more and smaller boxes)
        tma_box(at + kWeightBytes, &tmap, fb, kb * kTileCols, it.row0, leader);
        tma_box(at + kWeightBytes + g.bt * 128, &tmap, fb, kb * kTileCols + 64, it.row0, leader);
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
      ok = wait_parked(dempty0 + 8 * db, d_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
      for (int kb = kb0; ok && kb < kb1; ++kb) {
        // (the warps that filled the buffer have waited for the stage, rows of x and all)
        ok = wait_parked(afull0 + 8 * ab, a_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_FULL);
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
        if (++ab == a_bufs) ab = 0, a_phase ^= 1;
      }
      if (!ok) break;
      commit(dfull0 + 8 * db, leader);
      if (++db == g.d_bufs) db = 0, d_phase ^= 1;
    }
  } else if (warp < 6) {
    write_results<SPLIT, false>(g, first_tile, i0, i_step, items, kb0 == 0, tmem, dfull0, dempty0, reinterpret_cast<float*>(smem), staging, 0, 1, warp & 3,
                         lane, abort_flag, status);
  } else {
    // ---- codes -> bf16 in tensor memory: sets of four warps take the blocks in turn, a set a whole block
    const int q = warp & 3, set = (warp - 6) >> 2, r = q * 32 + lane;
    const uint32_t dst0 = tmem_a + (static_cast<uint32_t>(q * 32) << 16);
    // every block of the CTA's items in turn
    const int blocks = (kb1 - kb0) * (i0 < items ? (items - i0 + i_step - 1) / i_step : 0);
    int stage = set % g.stages, ab = set % a_bufs;
    uint32_t phase = (set / g.stages) & 1, a_phase = 1 ^ ((set / a_bufs) & 1);
    for (int n = set; n < blocks; n += kSets) {
      const uint32_t at = smem_u32(smem) + stage * stage_bytes;
      // First the buffer: that the product of a_bufs blocks ago is done says that every block up to it has been loaded, and with at
      // least as many stages as buffers so has the one that the stage held before. Loads end in any order, and the other set's may be
      // the later one: a wait for a phase whose predecessor is still open would return at once, with the stage half full.
      if (!wait_parked(aempty0 + 8 * ab, a_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY)) break;
      tc_fence_after_sync();
      if (!wait_parked(full0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL)) break;
      uint32_t code[4][4], p;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(code[h][0]), "=r"(code[h][1]), "=r"(code[h][2]), "=r"(code[h][3])
                     : "r"(at + r * 16 + h * (kTileRows * 16)));
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(p) : "r"(at + kCodeBytes + r * 4));
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t p2 = mx4_power2(p, h);
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t y[4];
          mx4_word(code[h][j], p2, shift, y);
#pragma unroll
          for (int v = 0; v < 4; ++v) o[4 * j + v] = y[v];
        }
        tmem_st_32x32b_x16(dst0 + ab * 64 + h * 16, o);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(afull0 + 8 * ab);
      for (ab += kSets; ab >= a_bufs; ab -= a_bufs) a_phase ^= 1;
      for (stage += kSets; stage >= g.stages; stage -= g.stages) phase ^= 1;
    }
  }

  if constexpr (SPLIT) {
    // Every thread of every CTA passes both barriers, also after a failed wait (all other waits are bounded).
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2) add_ranges(g, i0, smem_u32(smem), static_cast<int>(threadIdx.x) - 64, kThreads - 64, abort_flag);
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

int launch_product(const void* x, int64_t ldx, int x_rows, int K, const void* w, TileArgs g, int64_t items, int* status,
                   cudaStream_t stream) {
  static bool configured[64] = {};
  if (!pxl_host::allow_smem(configured, gemm_mx4_kernel<false>, gemm_mx4_kernel<true>)) return PXL_ERR_CUDA;
  if (items > 0x7fffffff) items = 0x7fffffff;
  const int sms = pxl_host::num_sms();
  // two CTAs per SM where their tiles are narrow: 256 columns of tensor memory and half of the shared memory each
  const bool two = g.bt <= 64;
  const int slots = two ? 2 * sms : sms;
  g.d_cols = pxl::ceil_div(g.bt, 32) * 32;
  g.d_bufs = !two && g.d_cols <= 192 ? 2 : 1;
  int a_bufs = ((two ? 256 : 512) - g.d_bufs * g.d_cols) / 64;
  if (a_bufs > kMaxBufs) a_bufs = kMaxBufs;
  pxl_host::split_k(g, items, slots, 12, gemm_mx4_kernel<true>, kThreads);
  const int stage_bytes = kWeightBytes + g.bt * 256, rest = 1024 + (g.offsets ? (g.experts + 1) * 4 : 0) + (g.splits == 1 && g.epi != PXL_EPI_NONE ? kStaging : 0);
  g.stages = ((two ? 113 * 1024 : pxl_host::kTileSmem) - 512 - rest) / stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  if (a_bufs > g.stages) a_bufs = g.stages;  // (see the warps that expand)
  if (a_bufs < kSets) return PXL_ERR_TOO_LARGE;
  int smem = rest + g.stages * stage_bytes;
  if (g.splits > 1 && smem < 1024 + g.bt * kPitch * 4) smem = 1024 + g.bt * kPitch * 4;
  CUtensorMap tmap;
  if (!pxl_host::make_tmap_2d(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, x_rows, K, ldx, g.bt, 64)) return PXL_ERR_TENSORMAP;
  return pxl_host::launch_tiles(gemm_mx4_kernel<false>, gemm_mx4_kernel<true>, g, static_cast<int>(items), slots, kThreads, smem, stream,
                                tmap, static_cast<const uint8_t*>(w), a_bufs, kMx4Shift, status);
}

// Width of the token tiles for more than 256 tokens. A tile's time is bound by the expansion up to 160 tokens (128, 144, 160: 0.89, 0.95,
// 1), and grows faster than its tokens beyond, where accumulators or buffers are fewer (176, 192, 224, 256: 1.15, 1.25, 1.48, 1.62), in
// the last case by results that no products hide. A last round that is not full takes about the mean of a round and of its part of one.
// 8192 x 4096 x 12288 in tiles of 160 tokens 660 us, 192 691, 256 621; 1000 x 8192 x 12288 185, 180, 159; 8192 x 24576 x 4096 1287,
// 1311, 1310.
int tile_tokens(int M, int n_blocks, int k_blocks) {
  const int sms = pxl_host::num_sms();
  int best = 160;
  int64_t least = INT64_MAX;
  for (int bt = 96; bt <= 256; bt += 16) {
    const int64_t tiles = static_cast<int64_t>(pxl::ceil_div(M, bt)) * n_blocks, rounds = (tiles + sms - 1) / sms;
    const int64_t time = bt <= 160 ? 8 * (bt + 126) : bt < 256 ? 15 * bt : 3670 + 3300 / k_blocks;
    const int64_t cost = (rounds * sms + tiles) * time;
    if (cost <= least) least = cost, best = bt;
  }
  return best;
}

bool epi_known(int epi, int N) {
  return epi == PXL_EPI_NONE || ((epi == PXL_EPI_SILU_MUL || epi == PXL_EPI_CLIP_GLU) && N % 128 == 0);
}

}  // namespace

PXL_EXPORT int pxl_gemm_mx4(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc,
                            const void* bias, const void* residual, int64_t ldr, int M, int N, int K, int epi, float limit,
                            int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 || !epi_known(epi, N) || !pxl_host::on16(x, 2 * ldx)) return PXL_ERR_INVALID_ARG;
  if (pxl_host::gemv_mx4_takes(M, N, K))
    return pxl_host::gemv_mx4(x, ldx, w, row_scale, C, ldc, bias, residual, ldr, M, N, K, epi, limit, stream);
  TileArgs g{};
  g.C = C, g.row_scale = row_scale, g.ldc = ldc, g.bias = static_cast<const bf16*>(bias);
  g.residual = static_cast<const bf16*>(residual), g.ldr = ldr, g.M = M, g.N = N, g.epi = epi, g.limit = limit;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kTileCols);
  // One tile for up to 256 tokens; in two, which expand all weights twice (us, one and two): 96 x 5120 x 25600 38 and 47, 203 60 and 75, 256
  // 66 and 86; 128 x 25600 x 5120 42 and 47, 203 64 and 64, 256 71 and 66; 128 x 12288 x 4096 19 and 25; 203 x 4096 x 4096 20.5 and 16.5.
  g.t_tiles = M <= 256 ? 1 : pxl::ceil_div(M, tile_tokens(M, g.n_blocks, g.k_blocks));
  g.bt = pxl::ceil_div(pxl::ceil_div(M, g.t_tiles), 16) * 16;
  // The SMs at work on 8 tiles of tokens share those and some 18 blocks of weights, from L2; with all tiles in one group x comes from
  // memory again for every few blocks (8192 rows of 24576 x 4096 1.45 -> 1.30 ms, of 4096 x 12288 0.90 -> 0.69; groups of 4 and 16: within
  // 2 % and 5 % of that). Rows of x that are 4-bit numbers themselves gain nothing (gemm_mx4_rows.cu: 422 -> 445 us for the former).
  g.t_group = 8;
  g.vec = pxl_host::on16(C, 2 * ldc) && (!residual || pxl_host::on16(residual, 2 * ldr));
  return launch_product(x, ldx, M, K, w, g, static_cast<int64_t>(g.n_blocks) * g.t_tiles, status, stream);
}

PXL_EXPORT int pxl_gemm_mx4_grouped(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc,
                                    int out_f32, const void* bias, int P, int E, int N, int K, const int* offsets, int epi,
                                    float limit, int* status, cudaStream_t stream) {
  if (P <= 0 || E <= 0 || E > kMaxExperts || N <= 0 || K <= 0 || K % 32 || !epi_known(epi, N) || !pxl_host::on16(x, 2 * ldx))
    return PXL_ERR_INVALID_ARG;
  TileArgs g{};
  g.C = C, g.row_scale = row_scale, g.ldc = ldc, g.out_f32 = out_f32, g.bias = static_cast<const bf16*>(bias);
  g.M = P, g.N = N, g.epi = epi, g.limit = limit;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kTileCols);
  g.offsets = offsets, g.experts = E;
  // One tile for an expert of an eighth more rows than the mean, up to 160. Lower tiles expand the weights of more experts twice (32
  // experts of 112 rows, 2880 x 2880, layer in us: 96 rows 347, 112 302, 128 252, 160 255), higher ones load rows that are not theirs
  // and have fewer stages (of 30 rows: 48 157, 64 157, 80 169, 128 175; of 512: 128 929, 160 877, 192 916).
  g.bt = 32;
  while (g.bt < 160 && 8ll * g.bt * E < 9ll * P) g.bt += 16;
  const int64_t items = static_cast<int64_t>(g.n_blocks) * (pxl::ceil_div(P, g.bt) + (P < E ? P : E));  // at most
  return launch_product(x, ldx, P, K, w, g, items, status, stream);
}
